"""MX FP4 operators (triton_chip_benchmarks_b200.mx): quantisation, products, a training step.

Values are compared with the numpy definition in 64 bits (oracle/mx.py).  Scales are
powers of two, so quantisation and dequantisation are exact up to their one
rounding: codes and scale bytes have to be equal.  Products of operands whose sums
are exact in fp32 have to be equal too (after the one rounding of the output).  Other
products may be off by what fp32 sums allow: a product of K terms t_i adds K values
that are exact in fp32 (code x code x power of two, or fp16 x code), each addition
off by at most 2^-23 of the running sum if it truncates, so

    |y - exact| <= K * 2^-23 * sum |t_i| + eps / 2 * |y|,   eps of the output's type.
"""

import numpy as np
import pytest
import torch

from oracle import mx as oracle_mx
from oracle import tensor as oracle_tensor
from triton_chip_benchmarks_b200 import _native, mx

BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32
gpu = pytest.mark.gpu


# ------------------------------------------------------------------ helpers
def f64(t: torch.Tensor) -> np.ndarray:
    return t.detach().cpu().double().numpy()


def rounded(y: np.ndarray, dtype: torch.dtype) -> torch.Tensor:
    return torch.from_numpy(np.ascontiguousarray(y)).to(dtype)


def same(a: torch.Tensor, b: torch.Tensor) -> bool:
    a, b = a.cpu(), b.cpu()
    return a.dtype == b.dtype and a.shape == b.shape and \
        bool(((a == b) | (a.isnan() & b.isnan())).all())


def parts(q: mx.MxTensor) -> tuple[np.ndarray, np.ndarray]:
    """Codes and padded scale codes of an MX tensor, on the host."""
    groups = (q.cols + 31) // 32
    return q.codes.cpu().numpy(), oracle_mx.unpack_scales(q.scales.cpu().numpy(), q.rows, groups)


def check_quantized(q: mx.MxTensor, x: np.ndarray, rule: str) -> None:
    codes, scales = oracle_mx.quantize(x, rule)
    got_codes, got_scales = parts(q)
    rows, groups = scales.shape
    assert np.array_equal(got_scales[:rows, :groups], scales)
    assert np.array_equal(got_codes, codes)
    padding = got_scales.copy()
    padding[:rows, :groups] = 127
    assert (padding == 127).all()


def mx_random(rows, cols, seed, low=124, high=131, device="cuda"):
    """An MX tensor of random codes with small scales, and its float64 values."""
    gen = np.random.default_rng(seed)
    groups = -(-cols // 32)
    codes = gen.integers(0, 16, (rows, groups * 32), dtype=np.uint8)
    codes[:, cols:] = 0
    scales = gen.integers(low, high, (rows, groups), dtype=np.uint8)
    packed = oracle_tensor.pack_e2m1_pairs(codes)
    q = mx.MxTensor.from_rows(torch.from_numpy(packed).to(device),
                              torch.from_numpy(scales).to(device), cols)
    return q, oracle_mx.dequantize(packed, scales, cols)


def activations(shape, dtype, seed, spread=1.0):
    gen = torch.Generator().manual_seed(seed)
    x = torch.randn(shape, generator=gen) * torch.exp(spread * torch.randn(shape[-1], generator=gen))
    return x.to(dtype)


def check_product(y: torch.Tensor, a: np.ndarray, b: np.ndarray, bias=None) -> None:
    exact = a @ b.T
    terms = np.abs(a) @ np.abs(b).T
    if bias is not None:
        exact, terms = exact + bias, terms + np.abs(bias)
    k = a.shape[1] + (bias is not None)
    bound = k * 2.0**-23 * terms + torch.finfo(y.dtype).eps / 2 * np.abs(exact) * (1 + 2.0**-8) \
        + torch.finfo(y.dtype).smallest_normal * torch.finfo(y.dtype).eps
    assert (np.abs(f64(y) - exact) <= bound).all()


# ------------------------------------------------------------- the definition
def test_oracle_rounds_ties_to_even_codes():
    x = np.array([[4.0, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 0.0, -0.25, -0.75, -5.0, 7.9, -7.9]])
    codes, scales = oracle_mx.quantize(x, "floor")
    assert scales.tolist() == [[127]]
    assert oracle_mx.dequantize(codes, scales, 14).tolist() == \
        [[4, 0, 1, 1, 2, 2, 4, 4, 0, 0, -1, -4, 6, -6]]
    codes, scales = oracle_mx.quantize(x, "up")
    assert scales.tolist() == [[128]]
    assert oracle_mx.dequantize(codes, scales, 14).tolist() == \
        [[4, 0, 1, 1, 2, 2, 4, 4, 0, 0, -1, -4, 8, -8]]


def test_oracle_packed_layout_round_trip():
    gen = np.random.default_rng(0)
    for rows, groups in ((1, 1), (130, 17), (256, 8)):
        scales = gen.integers(0, 256, (rows, groups), dtype=np.uint8)
        full = oracle_mx.unpack_scales(oracle_tensor.pack_mx_scales(scales), rows, groups)
        assert np.array_equal(full[:rows, :groups], scales)


# ------------------------------------------------------------------ refusals
def test_entry_points_refuse_bad_arguments_before_a_device_is_touched(native):
    lib = native.load()
    p = 0x1000  # never dereferenced
    bad, unsupported = native.ERR_INVALID_ARGUMENT, native.ERR_UNSUPPORTED
    quantize = lib.tcb_mx_quantize
    bf16, rule = native.T_BF16, native.MX_FLOOR
    assert quantize(bf16, p, -1, 4, 4, rule, p, p, None, None, None) == bad
    assert quantize(bf16, p, 4, 4, 3, rule, p, p, None, None, None) == bad       # pitch below cols
    assert quantize(bf16, p, 4, 4, 4, 2, p, p, None, None, None) == bad          # rule
    assert quantize(bf16, p, 4, 4, 4, rule, None, None, None, None, None) == bad  # no output
    assert quantize(bf16, p, 4, 4, 4, rule, p, None, None, None, None) == bad    # codes, no scales
    assert quantize(bf16, p, 4, 4, 4, rule, p, p, None, p, None) == bad
    assert quantize(bf16, None, 4, 4, 4, rule, p, p, None, None, None) == bad
    assert quantize(bf16, p, 1 << 31, 4, 4, rule, p, p, None, None, None) == bad
    assert quantize(native.T_FP64, p, 4, 4, 4, rule, p, p, None, None, None) == unsupported
    assert quantize(bf16, p + 1, 4, 4, 4, rule, p, p, None, None, None) == native.ERR_ALIGNMENT
    assert quantize(bf16, p, 4, 4, 4, rule, p + 8, p, None, None, None) == native.ERR_ALIGNMENT
    assert quantize(bf16, None, 0, 4, 4, rule, p, p, None, None, None) == native.OK
    assert quantize(bf16, None, 4, 0, 0, rule, p, p, p, p, None) == native.OK
    dequantize = lib.tcb_mx_dequantize
    assert dequantize(bf16, p, p, 4, 4, p, 3, None) == bad
    assert dequantize(bf16, p, None, 4, 4, p, 4, None) == bad
    assert dequantize(native.T_INT8, p, p, 4, 4, p, 4, None) == unsupported
    assert dequantize(native.T_FP32, p, p, 4, 4, p + 2, 4, None) == native.ERR_ALIGNMENT
    assert dequantize(bf16, None, None, 0, 4, None, 4, None) == native.OK
    gemm = lib.tcb_mx_gemm
    assert gemm(p, p, p, p, None, bf16, p, 8, 4, 8, 0, None, None) == bad        # K = 0
    assert gemm(p, p, p, p, None, bf16, p, 7, 4, 8, 32, None, None) == bad       # pitch below N
    assert gemm(p, None, p, p, None, bf16, p, 8, 4, 8, 32, None, None) == bad
    assert gemm(p, p, p, p, None, native.T_TF32, p, 8, 4, 8, 32, None, None) == unsupported
    assert gemm(p, p, p + 4, p, None, bf16, p, 8, 4, 8, 32, None, None) == native.ERR_ALIGNMENT
    assert gemm(None, None, None, None, None, bf16, None, 8, 0, 8, 32, None, None) == native.OK
    linear, none = lib.tcb_mx_linear, (None, 0, None, None)
    assert linear(bf16, p, 31, p, p, None, bf16, p, 8, 1, 8, 32, *none) == bad  # pitch below K
    assert linear(bf16, p, 32, p, p, None, bf16, None, 8, 1, 8, 32, *none) == bad
    assert linear(native.T_FP32, p, 32, p, p, None, bf16, p, 8, 1, 8, 32, *none) == unsupported
    assert linear(bf16, p, 32, p, p, None, native.T_INT8, p, 8, 1, 8, 32, *none) == unsupported
    assert linear(bf16, p, 32, p, p, p + 1, bf16, p, 8, 1, 8, 32, *none) == native.ERR_ALIGNMENT
    assert linear(bf16, None, 32, None, None, None, bf16, None, 8, 0, 8, 32, *none) == native.OK
    need = native.mx_linear_workspace_bytes(40, 1000)
    assert need > 0 and native.mx_linear_workspace_bytes(1, 1000) == 0
    assert linear(bf16, p, 1000, p, p, None, bf16, p, 8, 40, 8, 1000, p, need - 1, None, None) == bad
    assert linear(bf16, p, 1000, p, p, None, bf16, p, 8, 40, 8, 1000, None, need, None, None) == bad
    assert linear(bf16, p, 1000, p, p, None, bf16, p, 8, 40, 8, 1000, p + 16, need, None,
                  None) == native.ERR_ALIGNMENT
    with pytest.raises(native.TcbError):
        native.mx_linear_workspace_bytes(1, 0)


def test_host_tensors_and_wrong_codes_are_refused():
    x = torch.zeros(4, 64)
    with pytest.raises(ValueError, match="CUDA"):
        mx.quantize(x)
    with pytest.raises(TypeError):
        mx.quantize(x.double())
    with pytest.raises(ValueError, match="rule"):
        mx.quantize(x, rule="nearest")
    codes, scales = torch.zeros(4, 32, dtype=torch.uint8), torch.zeros(2048, dtype=torch.uint8)
    with pytest.raises(ValueError, match="CUDA"):
        mx.MxTensor(codes, scales, 4, 64)
    with pytest.raises(ValueError, match="codes"):
        mx.MxTensor(codes, scales, 4, 65)
    with pytest.raises(ValueError, match="scales"):
        mx.MxTensor(codes, scales[1:], 4, 64)
    with pytest.raises(TypeError):
        mx.MxTensor(codes.int(), scales, 4, 64)
    with pytest.raises(ValueError):
        mx.linear_forward(x, torch.zeros(8, 63))


@gpu
def test_shapes_types_and_strides_are_refused(cuda, native):
    x = torch.zeros(4, 64, device=cuda, dtype=BF16)
    q, w = mx.quantize(x), mx.quantize(torch.zeros(8, 96, device=cuda))
    with pytest.raises(ValueError):
        mx.matmul(q, w)  # 64 against 96 columns
    with pytest.raises(ValueError):
        mx.linear(x, w)
    with pytest.raises(TypeError):
        mx.linear(x.float(), q)
    with pytest.raises(TypeError):
        mx.matmul(q, q, dtype=torch.float64)
    with pytest.raises(TypeError):
        mx.matmul(q, q, bias=torch.zeros(4, device=cuda), dtype=BF16)
    with pytest.raises(ValueError):
        mx.matmul(q, q, bias=torch.zeros(5, device=cuda, dtype=BF16))
    with pytest.raises(ValueError):
        mx.matmul(q, q, out=torch.zeros(4, 5, device=cuda, dtype=BF16))
    with pytest.raises(ValueError):
        mx.matmul(q, q, out=torch.zeros(4, 4, device=cuda, dtype=BF16).t())
    with pytest.raises(ValueError):
        mx.matmul(q, q, out=torch.zeros(4, 4, dtype=BF16))
    with pytest.raises(ValueError):
        mx.quantize(torch.zeros(8, 64, device=cuda)[:, ::2].t()[::2])  # neither axis contiguous
    with pytest.raises(ValueError):
        mx.quantize(torch.zeros(1, 64, device=cuda).expand(4, 64))     # rows overlap
    with pytest.raises(ValueError):
        mx.quantize(torch.zeros(2, 3, 64, device=cuda).transpose(0, 1))
    with pytest.raises(ValueError):
        mx.linear(torch.zeros(64, 4, device=cuda, dtype=BF16).t(), q)
    empty = mx.quantize(torch.zeros(4, 0, device=cuda))
    with pytest.raises(ValueError):
        mx.matmul(empty, empty)
    y, saved = mx.linear_forward(torch.zeros(3, 32, device=cuda), torch.zeros(5, 32, device=cuda))
    with pytest.raises(ValueError):
        mx.linear_backward(torch.zeros(3, 4, device=cuda), saved)


# -------------------------------------------------------------- quantisation
@gpu
@pytest.mark.parametrize("rule", ["floor", "up"])
@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("shape", [(1, 1), (1, 32), (3, 31), (33, 257), (128, 128), (129, 130),
                                   (257, 96), (300, 1000)])
def test_quantize_both_axes(cuda, shape, dtype, rule):
    x = activations(shape, dtype, seed=shape[0] + shape[1], spread=2.0)
    d = x.to(cuda)
    check_quantized(mx.quantize(d, rule=rule), f64(x), rule)
    rows, cols = mx.quantize_pair(d, rule=rule)
    check_quantized(rows, f64(x), rule)
    check_quantized(cols, f64(x).T, rule)
    check_quantized(mx.quantize(d.t(), rule=rule), f64(x).T, rule)  # a transposed view alone


@gpu
@pytest.mark.parametrize("rule", ["floor", "up"])
@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
def test_quantize_special_values(cuda, dtype, rule):
    info = torch.finfo(dtype)
    tiny = info.smallest_normal
    groups = [
        [0.0, -0.0], [6.0, 5.0, 3.5, 2.5, 1.75, 1.25, 0.75, 0.25, -0.25, -5.0], [7.5, -7.5, 8.0],
        [info.max, -info.max, info.max / 2], [tiny, -tiny, tiny / 2, tiny * 3],
        [tiny * info.eps, 0.0, -tiny * info.eps], [float("inf"), 1.0], [1.0, -float("inf")],
        [float("nan"), 2.0], [float("nan"), float("inf")], [1.0] * 32, [1.5, 1.5078125], [1.5],
        [2.0**-10 * v for v in (1, 1.5, 1.75, 3)],
    ]
    x = torch.zeros(len(groups), 32, dtype=torch.float64)
    for i, g in enumerate(groups):
        x[i, :len(g)] = torch.tensor(g, dtype=torch.float64)
    x = x.to(dtype)
    check_quantized(mx.quantize(x.to(cuda), rule=rule), f64(x), rule)
    check_quantized(mx.quantize_pair(x.t().contiguous().to(cuda), rule=rule)[1], f64(x), rule)


@gpu
def test_quantize_strides_offsets_and_leading_axes(cuda):
    base = activations((40, 300), BF16, seed=1).to(cuda)
    for view in (base[:, :100], base[:, 3:200], base[5:, 8:264], base[::2, :64], base[7, 1:90],
                 base[:, 3:200].t(), base[::3].t(), base.view(4, 10, 300), base.view(2, 5, 4, 300)[1]):
        flat = view.reshape(-1, view.shape[-1])
        check_quantized(mx.quantize(view), f64(flat), "floor")
        a, b = mx.quantize_pair(view)
        check_quantized(a, f64(flat), "floor")
        check_quantized(b, f64(flat).T, "floor")


@gpu
@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("start", range(8))
def test_quantize_rows_off_the_16_byte_boundaries(cuda, dtype, start):
    """Several tiles, from every start; the last value of X is the storage's last."""
    gen = torch.Generator().manual_seed(start)
    for pitch in (385, 390 + start, 404):
        rows, cols = 300, pitch - start
        base = torch.randn(rows * pitch, generator=gen).to(dtype)
        host = base.view(rows, pitch)[:, start:]
        x = base.cuda().view(rows, pitch)[:, start:]
        check_quantized(mx.quantize(x), f64(host), "floor")
        a, b = mx.quantize_pair(x)
        check_quantized(a, f64(host), "floor")
        check_quantized(b, f64(host).T, "floor")
        check_quantized(mx.quantize(x[:, :257]), f64(host[:, :257]), "floor")


@gpu
def test_status_words_are_refused_off_the_device(cuda):
    w, x = mx.quantize(torch.ones(8, 64, device="cuda")), torch.ones(2, 64, device="cuda", dtype=BF16)
    for call in (lambda s: mx.matmul(w, w, status=s), lambda s: mx.linear(x, w, status=s)):
        with pytest.raises(ValueError, match="status"):
            call(torch.zeros(1, dtype=torch.int32))
        with pytest.raises(TypeError, match="status"):
            call(torch.zeros(1, dtype=torch.int64, device="cuda"))
        status = torch.zeros(1, dtype=torch.int32, device="cuda")
        call(status)
        assert status.item() == 0


@gpu
def test_quantize_nothing(cuda):
    for shape in ((0, 64), (64, 0), (0, 0)):
        a, b = mx.quantize_pair(torch.zeros(shape, device=cuda))
        assert a.shape == shape and b.shape == shape[::-1]
        assert mx.dequantize(a).shape == shape


@gpu
@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
def test_dequantize_every_code_and_scale(cuda, dtype):
    codes = np.tile(np.arange(16, dtype=np.uint8), (256, 2))
    packed = oracle_tensor.pack_e2m1_pairs(codes)
    scales = np.arange(256, dtype=np.uint8)[:, None]
    q = mx.MxTensor.from_rows(torch.from_numpy(packed).to(cuda),
                              torch.from_numpy(scales).to(cuda), 32)
    exact = oracle_mx.dequantize(packed, scales, 32)
    with np.errstate(over="ignore"):
        assert same(mx.dequantize(q, dtype), rounded(exact, FP32).to(dtype))


@gpu
@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("shape", [(1, 1), (5, 37), (130, 256), (257, 1001)])
def test_dequantize_shapes_and_pitch(cuda, shape, dtype):
    q, values = mx_random(*shape, seed=sum(shape))
    expected = rounded(values, dtype)
    assert same(mx.dequantize(q, dtype), expected)
    for pitch, offset in ((shape[1] + 3, 1), ((shape[1] + 15) // 8 * 8, 0)):
        room = torch.full((shape[0], pitch + offset), 9.0, dtype=dtype, device=cuda)
        out = room[:, offset:offset + shape[1]]
        assert mx.dequantize(q, out=out) is out
        assert same(out, expected)
        assert (room[:, :offset] == 9).all() and (room[:, offset + shape[1]:] == 9).all()


# ------------------------------------------------------------------ products
SHAPES = [(1, 1, 1), (1, 128, 32), (1, 300, 1000), (7, 130, 33), (8, 513, 257), (9, 96, 512),
          (16, 1000, 4096), (17, 257, 96), (32, 384, 2080), (33, 40, 64), (64, 640, 512),
          (65, 128, 288), (128, 520, 1000), (129, 255, 31), (300, 513, 544), (520, 264, 2048)]


@gpu
@pytest.mark.parametrize("dtype", [FP32, BF16, FP16])
@pytest.mark.parametrize("m,n,k", SHAPES)
def test_matmul_is_exact_where_fp32_sums_are(cuda, m, n, k, dtype):
    # Terms are multiples of 2^-2 * 2^-4; their absolute values sum to below 2^18, so
    # every partial sum is exact in fp32 (24 bits).
    a, va = mx_random(m, k, seed=m + k, low=125, high=130)
    b, vb = mx_random(n, k, seed=n + 7 * k, low=125, high=130)
    bias = rounded(np.random.default_rng(m).integers(-8, 9, n) / 4.0, dtype)
    exact = va @ vb.T
    assert (np.abs(va) @ np.abs(vb).T).max() < 2.0**24 * 2.0**-6
    status = torch.zeros(1, dtype=torch.int32, device=cuda)
    assert same(mx.matmul(a, b, dtype=dtype, status=status), rounded(exact, FP32).to(dtype))
    got = mx.matmul(a, b, bias=bias.to(cuda), dtype=dtype, status=status)
    assert same(got, rounded(exact + f64(bias), FP32).to(dtype))
    assert status.item() == 0


@gpu
@pytest.mark.parametrize("m,n,k", [(1, 300, 1000), (16, 513, 4096), (40, 130, 8192), (300, 520, 3000)])
@pytest.mark.parametrize("dtype", [FP32, BF16, FP16])
def test_matmul_of_quantized_data(cuda, m, n, k, dtype):
    a = mx.quantize(activations((m, k), FP32, seed=1).to(cuda))
    b = mx.quantize((activations((n, k), FP32, seed=2) * 0.02).to(cuda), rule="up")
    bias = activations((n,), dtype, seed=3)
    va, vb = f64(mx.dequantize(a, FP32)), f64(mx.dequantize(b, FP32))
    check_product(mx.matmul(a, b, dtype=dtype), va, vb)
    check_product(mx.matmul(a, b, bias=bias.to(cuda), dtype=dtype), va, vb, f64(bias))


@gpu
@pytest.mark.parametrize("m", [3, 40, 300])
@pytest.mark.parametrize("dtype", [FP32, BF16])
def test_matmul_into_a_pitched_output(cuda, m, dtype):
    n, k = 200, 160
    a, va = mx_random(m, k, seed=1)
    b, vb = mx_random(n, k, seed=2)
    expected = rounded(va @ vb.T, FP32).to(dtype)
    for pitch, offset in ((n + 8, 0), (n + 8, 8), (n + 5, 1)):
        room = torch.full((m, pitch + offset), 9.0, dtype=dtype, device=cuda)
        out = room[:, offset:offset + n]
        mx.matmul(a, b, out=out)
        assert same(out, expected)
        assert (room[:, :offset] == 9).all() and (room[:, offset + n:] == 9).all()


@gpu
@pytest.mark.parametrize("m", [2, 200])
def test_nan_scales_reach_their_rows_only(cuda, m):
    n, k = 150, 96
    x = activations((m, k), FP32, seed=5)
    w = activations((n, k), FP32, seed=6)
    x[1, 40] = float("nan")
    w[149, 0] = float("inf")
    a, b = mx.quantize(x.to(cuda)), mx.quantize(w.to(cuda))
    y = mx.matmul(a, b, dtype=FP32).cpu()
    assert y[1].isnan().all() and y[:, 149].isnan().all()
    keep = torch.ones(m, n, dtype=torch.bool)
    keep[1], keep[:, 149] = False, False
    assert y[keep].isfinite().all()
    z = mx.linear(x.to(BF16).to(cuda), b).cpu()
    assert z[1].isnan().all() and z[:, 149].isnan().all() and z[keep].isfinite().all()


@gpu
def test_products_over_nothing(cuda):
    a, b = mx.quantize(torch.zeros(0, 64, device=cuda)), mx.quantize(torch.zeros(5, 64, device=cuda))
    assert mx.matmul(a, b).shape == (0, 5) and mx.matmul(b, a).shape == (5, 0)
    assert mx.linear(torch.zeros(0, 64, device=cuda, dtype=BF16), b).shape == (0, 5)
    assert mx.linear(torch.zeros(2, 0, 64, device=cuda, dtype=BF16), b).shape == (2, 0, 5)


# ------------------------------------------------------- 16-bit rows x MX weight
@gpu
@pytest.mark.parametrize("x_dtype", [BF16, FP16])
@pytest.mark.parametrize("m,n,k", [(1, 1, 1), (1, 128, 256), (1, 4096, 4096), (2, 300, 1000), (8, 513, 257),
                                   (9, 96, 512), (16, 200, 2056), (17, 257, 96), (31, 384, 2080),
                                   (33, 130, 264), (64, 640, 512), (65, 128, 288), (200, 255, 777)])
def test_linear_is_exact_where_fp32_sums_are(cuda, m, n, k, x_dtype):
    gen = torch.Generator().manual_seed(m + n + k)
    x = (torch.randint(-16, 17, (m, k), generator=gen) / 4).to(x_dtype)  # multiples of 1/4 to 4
    w, vw = mx_random(n, k, seed=n + k, low=125, high=130)
    # Terms are multiples of 2^-5; their absolute values sum to below 2^19.
    assert (np.abs(f64(x)) @ np.abs(vw).T).max() < 2.0**24 * 2.0**-5
    exact = f64(x) @ vw.T
    status = torch.zeros(1, dtype=torch.int32, device=cuda)
    for dtype in (x_dtype, FP32):
        bias = rounded(np.random.default_rng(m).integers(-8, 9, n) / 4.0, dtype)
        assert same(mx.linear(x.to(cuda), w, dtype=dtype, status=status), rounded(exact, FP32).to(dtype))
        got = mx.linear(x.to(cuda), w, bias=bias.to(cuda), dtype=dtype, status=status)
        assert same(got, rounded(exact + f64(bias), FP32).to(dtype))
    assert status.item() == 0


@gpu
@pytest.mark.parametrize("x_dtype", [BF16, FP16])
@pytest.mark.parametrize("m,n,k", [(1, 300, 8192), (5, 513, 4136), (48, 260, 3000)])
def test_linear_of_activations(cuda, m, n, k, x_dtype):
    x = activations((m, k), x_dtype, seed=k, spread=1.5)
    w = mx.quantize((activations((n, k), FP32, seed=2) * 0.02).to(cuda))
    vw = f64(mx.dequantize(w, FP32))
    for dtype in (x_dtype, FP32):
        # A value is off by at most 2^-23 of its group's largest, which the bound
        # holds K times over for every term.
        check_product(mx.linear(x.to(cuda), w, dtype=dtype), f64(x), vw)


@gpu
@pytest.mark.parametrize("scale", [2.0**-100, 2.0**-60, 1.0, 2.0**100])
def test_linear_of_very_small_and_large_bf16_rows(cuda, scale):
    # Powers of two change nothing but the exponent.
    x = activations((3, 512), BF16, seed=9)
    w, vw = mx_random(200, 512, seed=4)
    exact = rounded(f64(mx.linear(x.to(cuda), w, dtype=FP32)) * scale, FP32)
    got = mx.linear((x.double() * scale).to(BF16).to(cuda), w, dtype=FP32)
    assert same(got, exact)


@gpu
def test_linear_of_the_smallest_normal_rows(cuda):
    x = torch.randint(-4, 5, (3, 300), generator=torch.Generator().manual_seed(2)).double() * 2.0**-126
    w, vw = mx_random(140, 300, seed=4)
    got = mx.linear(x.to(BF16).to(cuda), w, dtype=FP32)
    assert same(got, rounded(x.numpy() @ vw.T, FP32))  # multiples of 2^-130, exact


@gpu
@pytest.mark.parametrize("rows", [2, 8, 40])
def test_linear_with_infinite_rows(cuda, rows):
    x = activations((4, 300), BF16, seed=3)
    x[1, 7], x[2, 9], x[3, 299] = float("inf"), float("nan"), -float("inf")
    x[1, 8] = 1e30
    x = x.repeat((rows + 3) // 4, 1)[:rows]
    w = mx.quantize(activations((70, 300), FP32, seed=8).to(cuda))
    vw = f64(mx.dequantize(w, FP32))
    with np.errstate(invalid="ignore"):
        exact = f64(x) @ vw.T
    got = f64(mx.linear(x.to(cuda), w, dtype=FP32))
    assert np.array_equal(np.isnan(got), np.isnan(exact))
    infinite = np.isinf(exact)
    assert np.array_equal(got[infinite], exact[infinite]) and infinite.any()
    assert np.isfinite(got[0]).all()


@gpu
def test_linear_strides_offsets_and_leading_axes(cuda):
    w, vw = mx_random(130, 200, seed=4)
    base = (torch.randint(-8, 9, (24, 420), generator=torch.Generator().manual_seed(0)) / 4).to(BF16)
    d = base.to(cuda)
    for view, host in ((d[:, :200], base[:, :200]), (d[:, 3:203], base[:, 3:203]),
                       (d[::2, 8:208], base[::2, 8:208]), (d[5, 1:201], base[5, 1:201]),
                       (d.view(2, 12, 420)[:, :, 4:204], base.view(2, 12, 420)[:, :, 4:204])):
        exact = f64(host.reshape(-1, 200)) @ vw.T
        got = mx.linear(view, w)
        assert got.shape == (*view.shape[:-1], 130)
        assert same(got.reshape(-1, 130), rounded(exact, FP32).to(BF16))
    room = torch.full((24, 140), 9.0, dtype=BF16, device=cuda)
    mx.linear(d[:, :200], w, out=room[:, 4:134])
    assert same(room[:, 4:134], rounded(f64(base[:, :200]) @ vw.T, FP32).to(BF16))
    assert (room[:, :4] == 9).all() and (room[:, 134:] == 9).all()


# ------------------------------------------------------------- a training step
@gpu
@pytest.mark.parametrize("rule", ["floor", "up"])
@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("tokens,inner,outer", [(1, 32, 32), (5, 40, 70), (77, 160, 136), (300, 257, 130)])
def test_linear_step(cuda, tokens, inner, outer, dtype, rule):
    x, w = activations((tokens, inner), dtype, 1), (activations((outer, inner), FP32, 2) * 0.1).to(dtype)
    dy = (activations((tokens, outer), FP32, 3) * 0.1).to(dtype)
    y, saved = mx.linear_forward(x.to(cuda), w.to(cuda), rule=rule)
    dx, dw = mx.linear_backward(dy.to(cuda), saved)
    assert (y.dtype, dx.dtype, dw.dtype) == (dtype,) * 3
    assert dx.shape == x.shape and dw.shape == w.shape

    def q(v):
        return oracle_mx.dequantize(*oracle_mx.quantize(v, rule), v.shape[1])

    check_product(y, q(f64(x)), q(f64(w)))
    check_product(dx, q(f64(dy)), q(f64(w).T))
    check_product(dw, q(f64(dy).T), q(f64(x).T))
    only_dx, none = mx.linear_backward(dy.to(cuda), saved, need_dw=False)
    assert none is None and same(only_dx, dx)
    none, only_dw = mx.linear_backward(dy.to(cuda), saved, need_dx=False)
    assert none is None and same(only_dw, dw)


@gpu
def test_linear_gradients_are_the_differences_of_the_forward_pass(cuda):
    # Values that MX FP4 holds along both axes (codes with unit scale, a 4 in every
    # group pinning the scale), so the forward pass is linear between them and
    # L = sum(dy * y) has exact differences: moving one value by 1 moves L by its
    # gradient.
    gen = np.random.default_rng(0)

    def values(rows, cols):
        v = gen.choice([0.0, 1.0, 2.0, -1.0, -2.0], (rows, cols))
        v[::8, :], v[:, ::8] = 4.0, 4.0
        return torch.from_numpy(v).float()

    x, w, dy = values(64, 96), values(32, 96), values(64, 32)
    y, saved = mx.linear_forward(x.to(cuda), w.to(cuda))
    dx, dw = mx.linear_backward(dy.to(cuda), saved)

    def loss(x, w):
        return (dy.double() * mx.linear_forward(x.to(cuda), w.to(cuda))[0].cpu().double()).sum().item()

    at = loss(x, w)
    for i, j in ((1, 1), (17, 34), (63, 95)):
        moved = x.clone()
        moved[i, j] += 1
        assert loss(moved, w) - at == dx[i, j].item()
    for i, j in ((1, 1), (17, 34), (31, 95)):
        moved = w.clone()
        moved[i, j] += 1
        assert loss(x, moved) - at == dw[i, j].item()


@gpu
def test_linear_step_without_rows(cuda):
    w = torch.ones(8, 64, device=cuda)
    y, saved = mx.linear_forward(torch.zeros(2, 0, 64, device=cuda), w)
    dx, dw = mx.linear_backward(torch.zeros(2, 0, 8, device=cuda), saved)
    assert y.shape == (2, 0, 8) and dx.shape == (2, 0, 64)
    assert dw.shape == (8, 64) and (dw == 0).all()


# ------------------------------------------------------------- used together
@gpu
def test_a_layer_and_its_decoding_captured_and_replayed(cuda):
    """Quantise a weight once; prefill with MX activations, decode with 16-bit rows,
    take a training step: in one graph, replayed on other inputs, as eagerly."""
    w = (activations((264, 520), FP32, 1) * 0.05).to(BF16).to(cuda)
    x, dy = torch.empty(70, 520, dtype=BF16, device=cuda), torch.empty(70, 264, dtype=BF16, device=cuda)
    weight = mx.quantize(w)

    def step():
        prefill = mx.matmul(mx.quantize(x), weight)
        token = mx.linear(x[-1:], weight)
        y, saved = mx.linear_forward(x, w)
        dx, dw = mx.linear_backward(dy, saved)
        return prefill, token, y, dx, dw

    def fill(seed):
        x.copy_(activations((70, 520), BF16, seed))
        dy.copy_(activations((70, 264), BF16, seed + 1))

    fill(10)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    for seed in (20, 30):
        fill(seed)
        graph.replay()
        torch.cuda.synchronize()
        for got, eager in zip(captured, step()):
            assert same(got, eager)
        assert same(captured[0], captured[2])  # the same product twice


@gpu
def test_two_streams_at_once_give_the_same_results(cuda):
    weights = [mx_random(700, 1024, seed=s)[0] for s in (1, 2)]
    xs = [activations((m, 1024), BF16, m).to(cuda) for m in (1, 40)]
    alone = [mx.linear(x, w) for x, w in zip(xs, weights)]
    products = [mx.matmul(mx.quantize(x), w) for x, w in zip(xs, weights)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in xs]
    for _ in range(5):
        got = []
        for s, x, w in zip(streams, xs, weights):
            with torch.cuda.stream(s):
                got.append((mx.linear(x, w), mx.matmul(mx.quantize(x), w)))
        torch.cuda.synchronize()
        for (y, z), a, p in zip(got, alone, products):
            assert same(y, a) and same(z, p)


@gpu
@pytest.mark.parametrize("m", [1, 5, 40])
def test_products_follow_the_kernels_before_them(cuda, m):
    """A weight written right before the product that reads it, a workspace and outputs
    that the next call reuses: results as with everything waited for."""
    n = k = 4096
    raw = [torch.randn(n, k, device=cuda, dtype=FP32) for _ in range(3)]
    xs = [activations((m, k), BF16, seed).to(cuda) for seed in range(3)]
    waited = []
    for i in range(9):
        w = mx.quantize(raw[i % 3])
        torch.cuda.synchronize()
        waited.append(mx.linear(xs[i // 3], w))
        torch.cuda.synchronize()
    w = mx.MxTensor.empty_on(raw[0], n, k)
    got = []
    for i in range(9):
        _native.mx_quantize(_native.T_FP32, raw[i % 3], n, k, k, _native.MX_FLOOR, w.codes, w.scales)
        got.append(mx.linear(xs[i // 3], w))
    for a, b in zip(got, waited):
        assert torch.equal(a, b)


@gpu
@pytest.mark.parametrize("m", [1, 4, 40, 130])
@pytest.mark.parametrize("k", [512, 2048])
def test_chains_of_layers_that_reuse_two_buffers(cuda, m, k):
    """Each call reads what the one before wrote, in a buffer that the one before that
    read: as with everything waited for, eagerly and in a graph."""
    weights = [mx.quantize(torch.randn(k, k, device=cuda) * k ** -0.5) for _ in range(3)]
    start = activations((m, k), BF16, m).to(cuda)

    def chain(waiting):
        buffers = [start.clone(), torch.empty_like(start)]
        codes = mx.MxTensor.empty_on(start, m, k)
        for i in range(24):
            x, y = buffers[i % 2], buffers[1 - i % 2]
            if i % 3 == 2:
                _native.mx_quantize(_native.T_BF16, x, m, k, k, _native.MX_FLOOR, codes.codes, codes.scales)
                if waiting:
                    torch.cuda.synchronize()
                mx.matmul(codes, weights[i % 3], out=y)
            elif m <= 40:
                mx.linear(x, weights[i % 3], out=y)
            else:
                mx.matmul(mx.quantize(x), weights[i % 3], out=y)
            if waiting:
                torch.cuda.synchronize()
        return buffers[0]

    waited = chain(True)
    assert waited.isfinite().all() and waited.abs().max() > 0
    for _ in range(3):
        assert torch.equal(chain(False), waited)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = chain(False)
    for _ in range(5):
        graph.replay()
    assert torch.equal(captured, waited)


@gpu
def test_offsets_past_32_bits(cuda):
    """More than 2^32 values and 2^31 bytes of codes: the last rows are as those of a
    small tensor."""
    rows, cols, tail = 140000, 32768, 200
    if torch.cuda.mem_get_info()[0] < 30 << 30:
        pytest.skip("needs 30 GB of device memory")
    x = torch.zeros(rows, cols, dtype=BF16, device=cuda)
    x[-tail:] = torch.randn(tail, cols, device=cuda).to(BF16)
    q = mx.quantize(x)
    small = mx.quantize(x[-tail:].contiguous())
    assert torch.equal(q.codes[-tail:], small.codes)
    assert (q.codes[-tail - 100:-tail] == 0).all()
    y = torch.full_like(x, 9.0)
    del x
    mx.dequantize(q, out=y)
    assert torch.equal(y[-tail:], mx.dequantize(small))
    assert (y[rows // 2:-tail] == 0).all()
    del y
    # The sums may be split otherwise over K in the small product: both are held to the
    # exact one.
    values = f64(mx.dequantize(small, FP32))
    for m in (1, 5, 20):
        a = activations((m, cols), BF16, m).to(cuda)
        check_product(mx.linear(a, q)[:, -tail:], f64(a), values)
    a = mx.quantize(activations((3, cols), BF16, 9).to(cuda))
    va = f64(mx.dequantize(a, FP32))
    check_product(mx.matmul(a, q)[:, -tail:], va, values)
    check_product(mx.matmul(q, a)[-tail:], values, va)


def test_call_module_refuses_what_the_library_does_not_take(native):
    calls = native.calls()
    p = 0x1000  # never dereferenced
    assert calls.tcb_mx_quantize(0, p, 4, 4, 3, 0, p, p, None, None, None) == native.ERR_INVALID_ARGUMENT
    assert calls.tcb_mx_gemm(p, p, p, p, None, 0, p, 8, 1 << 32, 8, 32, None, None) == \
        native.ERR_INVALID_ARGUMENT  # a size past int is not cut off
    with pytest.raises(TypeError):
        calls.tcb_mx_dequantize(0, p, p)
    with pytest.raises(TypeError):
        calls.tcb_mx_quantize(0, "x", 4, 4, 4, 0, p, p, None, None, None)
    with pytest.raises(OverflowError):
        calls.tcb_mx_quantize(0, 1 << 70, 4, 4, 4, 0, p, p, None, None, None)


@gpu
@pytest.mark.parametrize("dtype", [FP32, BF16])
@pytest.mark.parametrize("n,pitch", [(4096, 4096), (4099, 4099), (4099, 4102), (4100, 4104)])
def test_matmul_with_more_tiles_than_pairs(cuda, n, pitch, dtype):
    """Several tiles a CTA pair, with rows of C on and off 16-byte boundaries."""
    m, k = 2400, 96
    a, va = mx_random(m, k, seed=1)
    b, vb = mx_random(n, k, seed=2)
    bias = rounded(np.random.default_rng(3).integers(-8, 9, n) / 4.0, dtype)
    exact = va @ vb.T
    room = torch.full((m, pitch), 9.0, dtype=dtype, device=cuda)
    mx.matmul(a, b, out=room[:, :n])
    assert same(room[:, :n], rounded(exact, FP32).to(dtype)) and (room[:, n:] == 9).all()
    mx.matmul(a, b, out=room[:, :n], bias=bias.to(cuda))
    assert same(room[:, :n], rounded(exact + f64(bias), FP32).to(dtype)) and (room[:, n:] == 9).all()


@gpu
def test_linear_with_more_tiles_than_pairs(cuda):
    m, n, k = 300, 2500, 96
    gen = torch.Generator().manual_seed(0)
    x = (torch.randint(-16, 17, (m, k), generator=gen) / 4).to(BF16)
    w, vw = mx_random(n, k, seed=5)
    assert same(mx.linear(x.to(cuda), w), rounded(f64(x) @ vw.T, FP32).to(BF16))


@gpu
@pytest.mark.parametrize("x_dtype", [BF16, FP16])
@pytest.mark.parametrize("m,n,k", [(17, 1, 40), (32, 130, 257), (33, 513, 300), (130, 1000, 130),  # column tiles
                                   (17, 19001, 70), (33, 18945, 300), (130, 2200, 130)])  # CTA pairs
def test_linear_of_more_rows_than_a_column_tile(cuda, m, n, k, x_dtype):
    gen = torch.Generator().manual_seed(m + n + k)
    x = (torch.randint(-16, 17, (m, k), generator=gen) / 4).to(x_dtype)
    w, vw = mx_random(n, k, seed=n + k, low=125, high=130)
    # Terms are multiples of 2^-5; their absolute values sum to below 2^19.
    assert (np.abs(f64(x)) @ np.abs(vw).T).max() < 2.0**24 * 2.0**-5
    exact = f64(x) @ vw.T
    for dtype in (x_dtype, FP32):
        bias = rounded(np.random.default_rng(m).integers(-8, 9, n) / 4.0, dtype)
        got = mx.linear(x.to(cuda), w, bias=bias.to(cuda), dtype=dtype)
        assert same(got, rounded(exact + f64(bias), FP32).to(dtype))
    # Into a pitched output, whose gap stays as it is.
    wide = torch.full((m, n + 5), 7.0, dtype=x_dtype, device=cuda)
    mx.linear(x.to(cuda), w, out=wide[:, :n])
    assert same(wide[:, :n], rounded(exact, FP32).to(x_dtype)) and (wide[:, n:] == 7).all()
    # Infinities and NaN in their rows alone.
    x[0, 1], x[m - 1, k - 1], x[16, 5] = float("inf"), -float("inf"), float("nan")
    with np.errstate(invalid="ignore"):
        exact = f64(x) @ vw.T
    assert same(mx.linear(x.to(cuda), w, dtype=FP32), rounded(exact, FP32))


@gpu
def test_linear_of_many_rows_follows_the_kernels_before_it(cuda):
    """Column tiles, and pairs, whose weight and workspace the calls before have just written."""
    for m, n, k in ((40, 1024, 2048), (40, 19200, 512)):
        raw = [torch.randn(n, k, device=cuda) for _ in range(2)]
        xs = [activations((m, k), BF16, seed).to(cuda) for seed in range(2)]
        waited = []
        for i in range(6):
            w = mx.quantize(raw[i % 2])
            torch.cuda.synchronize()
            waited.append(mx.linear(xs[i // 3], w))
            torch.cuda.synchronize()
        w = mx.MxTensor.empty_on(raw[0], n, k)
        got = []
        for i in range(6):
            _native.mx_quantize(_native.T_FP32, raw[i % 2], n, k, k, _native.MX_FLOOR, w.codes, w.scales)
            got.append(mx.linear(xs[i // 3], w))
        for a, b in zip(got, waited):
            assert torch.equal(a, b)
