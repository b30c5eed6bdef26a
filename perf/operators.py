"""Workloads of the microscaled 4-bit (MX FP4) operators, in plain and in native form.

A value of an MX FP4 tensor is an E2M1 code (0, 0.5, 1, 1.5, 2, 3, 4 or 6 with a
sign) times a power of two that 32 neighbours along the inner axis share.  The
operators are

  quantize       rows of a bf16, fp16 or fp32 tensor to codes and scales, along the
                 rows only or along both axes in one pass, and dequantize back;
  matmul         the product of two MX tensors, A [M][K] . B [N][K]^T;
  linear         bf16 or fp16 rows times an MX weight (few rows: decoding);
  linear_forward / linear_backward
                 a linear layer's training step on MX products: y, dx and dw.

``own = False`` computes them with elementary torch operations, ``own = True`` with
``triton_chip_benchmarks_b200.mx``.  A quantised tensor is returned as the values it
stands for.
"""

import torch

own = False

GROUP = 32
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}


# ------------------------------------------------------------------ the cases
def listed():
    return [
        # One token's activations before a quantised product: latency alone.
        dict(name="quantize 1x4096 bf16", op="quantize", rows=1, cols=4096, dtype="bf16", rule="floor"),
        # A long prefill's activations, or a weight that is quantised once.
        dict(name="quantize 8192x8192 bf16", op="quantize", rows=8192, cols=8192, dtype="bf16", rule="floor"),
        # Ragged both ways, in fp32: a master weight with the scale rounded up.
        dict(name="pair 4099x2072 fp32 up", op="pair", rows=4099, cols=2072, dtype="fp32", rule="up"),
        # A training batch's activations, once along each axis.
        dict(name="pair 8192x4096 bf16", op="pair", rows=8192, cols=4096, dtype="bf16", rule="floor"),
        # The size of the framework's own FP4 product row.
        dict(name="matmul 8192x8192x8192 bf16", op="matmul", m=8192, n=8192, k=8192, dtype="bf16", bias=False),
        # Ragged sizes in all three directions, a bias, full-precision output.
        dict(name="matmul 1000x4104x2072 fp32", op="matmul", m=1000, n=4104, k=2072, dtype="fp32", bias=True),
        # A small decoding batch with quantised activations: the weight is what counts.
        dict(name="matmul 16x8192x8192 bf16", op="matmul", m=16, n=8192, k=8192, dtype="bf16", bias=False),
        # One token through a projection: latency.
        dict(name="linear 1x4096x4096 bf16", op="linear", m=1, n=4096, k=4096, dtype="bf16", bias=False),
        # One token through a wide projection: the weight's bytes.
        dict(name="linear 1x16384x8192 bf16", op="linear", m=1, n=16384, k=8192, dtype="bf16", bias=False),
        # A decoding batch with odd sizes and a bias.
        dict(name="linear 33x5000x4136 fp16", op="linear", m=33, n=5000, k=4136, dtype="fp16", bias=True),
        # A training step of one linear layer.
        dict(name="train 4096x4096x4096 bf16", op="train", m=4096, n=4096, k=4096, dtype="bf16", rule="floor"),
        # The same on a ragged batch with fp32 master weights.
        dict(name="train 777x1056x2016 fp32", op="train", m=777, n=1056, k=2016, dtype="fp32", rule="up"),
    ]


def draw(rng):
    def size(low, high):
        return max(low, min(high, int(low * (high / low) ** rng.random())))

    op = rng.choice(["quantize", "pair", "matmul", "linear", "train"])
    if op in ("quantize", "pair"):
        rows = size(1 if op == "quantize" else 16, 16384)
        return dict(op=op, rows=rows, cols=size(32, min(16384, (1 << 26) // rows)),
                    dtype=rng.choice(["bf16", "bf16", "fp16", "fp32"]), rule=rng.choice(["floor", "up"]))
    if op == "matmul":
        return dict(op=op, m=size(1, 8192), n=size(64, 8192), k=size(64, 8192),
                    dtype=rng.choice(["bf16", "fp16", "fp32"]), bias=rng.random() < 0.3)
    if op == "linear":
        return dict(op=op, m=size(1, 64), n=size(256, 16384), k=size(256, 16384),
                    dtype=rng.choice(["bf16", "fp16"]), bias=rng.random() < 0.3)
    return dict(op=op, m=size(64, 8192), n=size(128, 4608), k=size(128, 4608),
                dtype=rng.choice(["bf16", "fp16", "fp32"]), rule=rng.choice(["floor", "up"]))


def _up(n, unit):
    return (n + unit - 1) // unit * unit


def _mx_bytes(rows, cols):
    return rows * _up(cols, GROUP) * 17 // 32  # half a byte a value, one byte a group


def work(case):
    op = case["op"]
    b = BYTES[case["dtype"]]
    if op in ("quantize", "pair"):
        # The input read; each quantised tensor written, read back, and its values written.
        r, c = case["rows"], case["cols"]
        total = r * c * b + 2 * _mx_bytes(r, c) + r * c * b
        if op == "pair":
            total += 2 * _mx_bytes(c, r) + r * c * b
        return dict(bytes=total, flops=0)
    m, n, k = case["m"], case["n"], case["k"]
    if op == "matmul":
        return dict(bytes=_mx_bytes(m, k) + _mx_bytes(n, k) + m * n * b + (n * b if case["bias"] else 0),
                    flops=2 * m * n * k)
    if op == "linear":
        return dict(bytes=m * k * b + _mx_bytes(n, k) + m * n * b + (n * b if case["bias"] else 0),
                    flops=2 * m * n * k)
    # x, w and dy read; y, dx and dw written.
    return dict(bytes=2 * b * (m * k + n * k + m * n), flops=6 * m * n * k)


# ------------------------------------------------------- plain form (32 bits)
def _quantize(x, rule):
    """Codes [rows][groups * 32] (one a byte) and scale exponents [rows][groups] of x's rows."""
    rows, cols = x.shape
    padded = _up(cols, GROUP)
    v = torch.zeros(rows, padded, dtype=torch.float32, device=x.device)
    v[:, :cols] = x
    v = v.view(rows, padded // GROUP, GROUP)
    top = v.abs().amax(-1)
    mantissa, exponent = torch.frexp(top)  # top = mantissa * 2^exponent, mantissa in [0.5, 1)
    e = exponent - 3
    if rule == "up":
        e = e + (mantissa > 0.75)  # 6 * 2^e holds the largest value
    e = torch.where(top == 0, torch.zeros_like(e), e).clamp(min=-127)
    v = torch.ldexp(v, -e.unsqueeze(-1))
    a = v.abs()
    step = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0))
    a = (torch.round(a / step) * step).clamp(max=6)  # round() takes halves to even
    code = torch.where(a < 2, a * 2, torch.where(a < 4, a + 2, a / 2 + 4)).to(torch.uint8)
    code = code + (v < 0).to(torch.uint8) * 8
    return code.view(rows, padded), e


_E2M1 = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]


def _values(code, e, cols):
    """The values that codes [rows][padded] and exponents [rows][groups] stand for, in fp32."""
    table = torch.tensor(_E2M1 + [-v for v in _E2M1], device=code.device)
    v = table[code.long()].view(code.shape[0], -1, GROUP)
    return torch.ldexp(v, e.unsqueeze(-1)).view(code.shape[0], -1)[:, :cols]


def _unpack(codes):
    return torch.stack((codes & 15, codes >> 4), -1).view(codes.shape[0], -1)


def _rounded(x, rule):
    return _values(*_quantize(x, rule), x.shape[1])


def _plain(state):
    case, op = state["case"], state["case"]["op"]
    if op in ("quantize", "pair"):
        x, rule = state["x"], case["rule"]
        rows = _rounded(x, rule).to(x.dtype)
        if op == "quantize":
            return rows
        return rows, _rounded(x.t(), rule).to(x.dtype)
    if op == "train":
        x, w, dy, rule = state["x"], state["w"], state["dy"], case["rule"]
        y = _rounded(x, rule) @ _rounded(w, rule).t()
        dx = _rounded(dy, rule) @ _rounded(w.t(), rule).t()
        dw = _rounded(dy.t(), rule) @ _rounded(x.t(), rule).t()
        return y.to(x.dtype), dx.to(x.dtype), dw.to(w.dtype)
    k = case["k"]
    if op == "matmul":
        a = _values(_unpack(state["a"]["codes"]), state["a"]["exponents"].int() - 127, k)
    else:
        a = state["x"].float()
    w = _values(_unpack(state["w"]["codes"]), state["w"]["exponents"].int() - 127, k)
    y = a @ w.t()
    if state["bias"] is not None:
        y = y + state["bias"].float()
    return y.to(DTYPES[case["dtype"]])


# ------------------------------------------------------------------- the calls
def _own(state):
    from triton_chip_benchmarks_b200 import mx

    case, op = state["case"], state["case"]["op"]
    if op == "quantize":
        return mx.dequantize(mx.quantize(state["x"], rule=case["rule"]), state["x"].dtype)
    if op == "pair":
        rows, cols = mx.quantize_pair(state["x"], rule=case["rule"])
        return mx.dequantize(rows, state["x"].dtype), mx.dequantize(cols, state["x"].dtype)
    if op == "train":
        y, saved = mx.linear_forward(state["x"], state["w"], rule=case["rule"])
        dx, dw = mx.linear_backward(state["dy"], saved)
        return y, dx, dw

    def tensor(t):
        return mx.MxTensor(t["codes"], t["scales"], t["rows"], t["cols"])

    if op == "matmul":
        return mx.matmul(tensor(state["a"]), tensor(state["w"]), bias=state["bias"],
                         dtype=DTYPES[case["dtype"]])
    return mx.linear(state["x"], tensor(state["w"]), bias=state["bias"])


def run(state):
    return _own(state) if own else _plain(state)


# ------------------------------------------------------------------ the inputs
def _activations(rows, cols, dtype, gen):
    """Normal values with channels of different sizes, a few of them large."""
    x = torch.randn(rows, cols, device="cuda", generator=gen)
    channel = torch.randn(cols, device="cuda", generator=gen)
    return (x * torch.exp(channel)).to(DTYPES[dtype])


def _packed(exponents):
    """The scale layout that the framework's MX FP4 product reads: rows to a multiple of
    256 and groups to one of 8 (padding 127), then 1 KiB a 128 rows and 8 groups: two
    halves of 4 groups, 32 lanes, the rows l, 32 + l, 64 + l, 96 + l, 4 bytes each."""
    rows, groups = exponents.shape
    full = torch.full((_up(rows, 256), _up(groups, 8)), 127, dtype=torch.uint8, device="cuda")
    full[:rows, :groups] = exponents
    s = full.view(full.shape[0] // 128, 4, 32, full.shape[1] // 8, 2, 4)
    return s.permute(0, 3, 4, 2, 1, 5).reshape(-1)


def _mx(x):
    """An MX tensor as a program keeps it, with its exponents by rows beside it."""
    code, e = _quantize(x.float(), "floor")
    exponents = (e + 127).to(torch.uint8)
    return dict(codes=code[:, 0::2] | (code[:, 1::2] << 4), scales=_packed(exponents),
                exponents=exponents, rows=x.shape[0], cols=x.shape[1])


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    op, dtype = case["op"], case["dtype"]
    if op in ("quantize", "pair"):
        return dict(case=case, x=_activations(case["rows"], case["cols"], dtype, gen))
    m, n, k = case["m"], case["n"], case["k"]
    w = torch.randn(n, k, device="cuda", generator=gen) * 0.02
    if op == "train":
        dy = torch.randn(m, n, device="cuda", generator=gen) * 0.01
        return dict(case=case, x=_activations(m, k, dtype, gen), w=w.to(DTYPES[dtype]), dy=dy.to(DTYPES[dtype]))
    bias = torch.randn(n, device="cuda", generator=gen).to(DTYPES[dtype]) if case["bias"] else None
    x = _activations(m, k, "fp32" if op == "matmul" else dtype, gen)
    if op == "matmul":
        return dict(case=case, a=_mx(x), w=_mx(w), bias=bias)
    return dict(case=case, x=x, w=_mx(w), bias=bias)


# ------------------------------------------------------- the definition, 64 bits
def _exact_rounded(x, rule):
    """x [rows][cols] with each group of 32 along a row on its MX FP4 grid."""
    rows, cols = x.shape
    v = torch.nn.functional.pad(x.double(), (0, _up(cols, GROUP) - cols)).view(rows, -1, GROUP)
    top = v.abs().amax(-1, keepdim=True)
    # The powers of two from a table: the largest one that is not above the top.
    powers = torch.tensor([2.0**i for i in range(-160, 130)], dtype=torch.float64, device=x.device)
    at = torch.bucketize(torch.where(top > 0, top, 1.0), powers, right=True) - 1 - 2
    if rule == "up":
        at = at + (top > 6 * powers[at])
    scale = powers[at.clamp(min=160 - 127)]
    grid = torch.tensor(_E2M1, dtype=torch.float64, device=x.device)
    middle = (grid[1:] + grid[:-1]) / 2
    a = (v.abs() / scale).contiguous()
    low, high = torch.bucketize(a, middle), torch.bucketize(a, middle, right=True)
    code = torch.where(low % 2 == 0, low, high)  # a tie goes to the even code
    code = torch.where(low == high, low, code)
    return (grid[code] * torch.sign(v) * scale).view(rows, -1)[:, :cols]


def _exact_values(t):
    code = torch.stack((t["codes"] % 16, t["codes"] // 16), -1).flatten(1).long()
    magnitude = code % 8
    value = torch.where(magnitude < 2, magnitude / 2.0,
                        (1 + (magnitude % 2) / 2.0) * (1 << (magnitude // 2).clamp(min=1)) / 2)
    value = torch.where(code >= 8, -value, value).double()
    powers = torch.tensor([2.0 ** (i - 127) for i in range(255)], dtype=torch.float64, device=code.device)
    return (value * powers[t["exponents"].long()].repeat_interleave(GROUP, 1))[:, :t["cols"]]


def exact(case, seed):
    state = prepare(case, seed)
    op = case["op"]
    if op in ("quantize", "pair"):
        rows = _exact_rounded(state["x"], case["rule"])
        return rows if op == "quantize" else (rows, _exact_rounded(state["x"].t(), case["rule"]))
    if op == "train":
        rule, x, w, dy = case["rule"], state["x"], state["w"], state["dy"]
        return (_exact_rounded(x, rule) @ _exact_rounded(w, rule).t(),
                _exact_rounded(dy, rule) @ _exact_rounded(w.t(), rule).t(),
                _exact_rounded(dy.t(), rule) @ _exact_rounded(x.t(), rule).t())
    a = _exact_values(state["a"]) if op == "matmul" else state["x"].double()
    y = a @ _exact_values(state["w"]).t()
    return y if state["bias"] is None else y + state["bias"].double()
