"""mx.linear on rows whose values differ widely in size, next to weights of zero.

A group's largest value may meet a weight of zero, and then nothing hides what the
smaller values lose.  Here every group's large value does: the small ones have full
mantissas, the weights unit scales, and the sums of the absolute terms (an eighth more,
for digits above the value that they begin) stay below 2^24 of their unit, so every
partial sum is exact in fp32 in any order and the results have to be equal.
"""

import numpy as np
import pytest
import torch

from oracle import mx as oracle_mx
from oracle import tensor as oracle_tensor
from triton_chip_benchmarks_b200 import mx

BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32
gpu = pytest.mark.gpu

# One and two rows, up to a column tile, more column tiles, pairs of CTAs.
SHAPES = [(1, 130, 300), (2, 300, 1000), (1, 64, 4100), (2, 129, 4100), (3, 130, 300), (16, 200, 1000),
          (9, 500, 4100), (17, 130, 300), (40, 260, 700), (130, 2200, 130), (17, 18950, 70)]


def weight(codes: np.ndarray, k: int):
    """An MX weight of unit scales from codes [n][whole groups], and its values."""
    packed = oracle_tensor.pack_e2m1_pairs(codes)
    scales = np.full((codes.shape[0], codes.shape[1] // 32), 127, dtype=np.uint8)
    q = mx.MxTensor.from_rows(torch.from_numpy(packed).cuda(), torch.from_numpy(scales).cuda(), k)
    return q, oracle_mx.dequantize(packed, scales, k)


def rows_and_weight(m, n, k, dtype, shift, share, seed):
    """Rows with values `shift` binary places above the others where the weights are
    zero: in every group (share 1), or in that share of the groups, next to two small
    values."""
    gen = np.random.default_rng(seed)
    groups = -(-k // 32)
    large = np.array([32 * g + gen.integers(min(32, k - 32 * g)) for g in range(groups)])
    codes = gen.integers(0, 16, (n, groups * 32), dtype=np.uint8)
    codes[:, k:] = 0
    codes[:, large] = 0
    low, unit = (129, 1.0) if dtype == BF16 else (1025, 2.0**-14)
    x = (2 * gen.integers(0, low // 2, (m, k)) + low) * unit * gen.choice([-1, 1], (m, k))  # full mantissas
    x *= gen.random((m, k)) < min(1.0, (400 if dtype == FP16 else 4000) / k)  # so that the sums fit 24 bits
    for g, at in enumerate(large):
        has = gen.random(m) < share
        if share < 1:
            inside = x[:, 32 * g:32 * g + 32]
            keep = np.argsort(gen.random(inside.shape), axis=1) < 2
            inside *= keep | ~has[:, None]
        x[:, at] = np.where(has, gen.choice([-1, 1], m) * 1.9375 * (low - 1) * unit * 2.0**shift, 0)
    host = torch.from_numpy(x).to(dtype)
    assert np.array_equal(host.double().numpy(), x)
    q, values = weight(codes, k)
    assert (np.abs(x) @ np.abs(values).T).max() * 9 / 8 < 2.0**24 * unit / 2
    return host, q, values


def equal(got: torch.Tensor, exact: np.ndarray) -> bool:
    return np.array_equal(got.cpu().double().numpy(), exact)


@gpu
@pytest.mark.parametrize("share", [1, 0.5, 0.03])
@pytest.mark.parametrize("dtype,shift", [(BF16, 7), (BF16, 14), (BF16, 17), (BF16, 24), (BF16, 100),
                                         (FP16, 7), (FP16, 12), (FP16, 19)])
@pytest.mark.parametrize("m,n,k", SHAPES)
def test_linear_keeps_small_values_beside_large_ones(cuda, m, n, k, dtype, shift, share):
    x, w, values = rows_and_weight(m, n, k, dtype, shift, share, seed=m + shift)
    exact = x.double().numpy() @ values.T
    status = torch.zeros(1, dtype=torch.int32, device=cuda)
    assert equal(mx.linear(x.to(cuda), w, dtype=FP32, status=status), exact)
    bias = torch.from_numpy(np.random.default_rng(0).integers(-8, 9, n) / 4.0).float().to(cuda)
    # One rounding behind the bias: their sum is exact in 32 bits more than fp32's.
    got = mx.linear(x.to(cuda), w, bias=bias, dtype=FP32, status=status)
    assert torch.equal(got.cpu(), torch.from_numpy(exact + bias.cpu().double().numpy()).float())
    assert status.item() == 0


@gpu
@pytest.mark.parametrize("dtype,shift", [(BF16, 24), (FP16, 19)])
@pytest.mark.parametrize("m,n,k", [(14, 140, 700), (15, 140, 700), (28, 140, 300), (29, 140, 300),  # full tiles
                                   (130, 4300, 8300), (20, 18950, 300)])  # pairs, more than 32 blocks of K
def test_linear_of_wide_rows_at_the_edges_of_tiles(cuda, m, n, k, dtype, shift):
    for share in (1, 0.03):
        x, w, values = rows_and_weight(m, n, k, dtype, shift, share, seed=m)
        assert equal(mx.linear(x.to(cuda), w, dtype=FP32), x.double().numpy() @ values.T)


@gpu
@pytest.mark.parametrize("m,n,k", [(1, 130, 40), (2, 130, 40), (5, 130, 40), (40, 300, 40), (20, 18950, 40)])
@pytest.mark.parametrize("power", [-97, -104, -110, -115, -120, -126])
def test_linear_of_full_mantissas_near_the_smallest_number(cuda, m, n, k, power):
    gen = np.random.default_rng(-power)
    x = gen.integers(129, 256, (m, k)) * 2.0 ** (power - 7) * gen.choice([-1, 1], (m, k))
    codes = gen.integers(0, 16, (n, 64), dtype=np.uint8)
    codes[:, k:] = 0
    w, values = weight(codes, k)
    host = torch.from_numpy(x).to(BF16)
    assert np.array_equal(host.double().numpy(), x)
    assert equal(mx.linear(host.to(cuda), w, dtype=FP32), x @ values.T)


@gpu
@pytest.mark.parametrize("m", [1, 4, 40])
def test_linear_of_subnormal_rows(cuda, m):
    gen = np.random.default_rng(m)
    k, n = 40, 130
    # Multiples of 2^-133 up to 2^-126, a few larger ones: exact in bf16.
    x = gen.integers(-127, 128, (m, k)) * 2.0**-133
    x[:, ::16] = gen.integers(1, 128, x[:, ::16].shape) * 2.0**-128
    codes = gen.integers(0, 16, (n, 64), dtype=np.uint8)
    codes[:, k:] = 0
    w, values = weight(codes, k)
    host = torch.from_numpy(x).to(BF16)
    assert np.array_equal(host.double().numpy(), x)
    assert equal(mx.linear(host.to(cuda), w, dtype=FP32), x @ values.T)


@gpu
@pytest.mark.parametrize("m,n", [(1, 140), (2, 140), (4, 140), (40, 140), (20, 18950)])
def test_linear_with_the_lowest_value_as_a_mask(cuda, m, n):
    """The lowest bf16 value: nothing where its weight is zero, itself where it is the
    only term and the weight is one, half of it at one half."""
    k = 300
    gen = np.random.default_rng(m)
    lowest = torch.finfo(BF16).min
    x = gen.integers(129, 256, (m, k)) * gen.choice([-1.0, 1.0], (m, k))
    x[:, 35] = lowest
    x[0, 64:96] = lowest  # a whole group
    codes = gen.integers(0, 16, (n, 320), dtype=np.uint8)
    codes[:, 300:] = 0
    codes[:, 35] = 0
    codes[:, 64:96] = 0
    codes[1] = codes[2] = 0
    codes[1, 35], codes[2, 35] = 2, 9  # 1 and -1/2
    w, values = weight(codes, k)
    got = mx.linear(torch.from_numpy(x).to(BF16).to(cuda), w, dtype=FP32)
    exact = x @ values.T
    assert (exact[:, 1] == lowest).all() and (exact[:, 2] == -lowest / 2).all()
    assert equal(got, exact)


@gpu
@pytest.mark.parametrize("m", [1, 2, 5, 40])
def test_linear_of_wide_rows_captured_and_replayed(cuda, m):
    """Rows with and without such values in turn through one graph: nothing stays
    behind from the ones before."""
    n, k = 260, 1000
    sets = [rows_and_weight(m, n, k, BF16, shift, share, seed=1)  # the same weight
            for shift, share in ((24, 1), (0, 1), (24, 0.03))]
    w, values = sets[0][1:]
    x = torch.empty(m, k, dtype=BF16, device=cuda)
    x.copy_(sets[1][0])
    mx.linear(x, w, dtype=FP32)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = mx.linear(x, w, dtype=FP32)
    for i in (0, 1, 2, 1, 0, 2):
        x.copy_(sets[i][0])
        graph.replay()
        assert equal(y, sets[i][0].double().numpy() @ values.T)
