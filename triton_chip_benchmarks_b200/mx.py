"""Microscaled 4-bit floating point (MX FP4) on torch tensors.

An :class:`MxTensor` stands for a matrix whose values are E2M1 codes times a power
of two shared by 32 neighbours of a row (OCP MX).  The operators run on the
tensors' device and on its current stream, allocate their outputs through torch unless
``out`` is given, never synchronise, and can be captured into a CUDA graph:

* :func:`quantize`, :func:`quantize_pair`, :func:`dequantize`: between torch tensors
  (bf16, fp16, fp32) and MX tensors, along one axis or both in one read;
* :func:`matmul`: ``a . b^T`` of two MX tensors;
* :func:`linear`: 16-bit rows times an MX weight (decoding);
* :func:`linear_forward`, :func:`linear_backward`: a linear layer's training step in
  MX products (both passes quantise their operands along the axis that the
  product sums over; gradients pass the rounding unchanged).

The operators are outside autograd: an output of one never requires a gradient, and
:func:`linear_backward` is called by hand (or by a ``torch.autograd.Function``).

Results are rounded once, from fp32 sums.  Arguments that an operator does not take
raise ``TypeError`` (types) or ``ValueError`` (shapes, strides, devices); what the
library itself refuses raises :class:`_native.TcbError`.
"""

from __future__ import annotations

from dataclasses import dataclass
import functools

import torch

from . import _native
from .validation import MX_GROUP_SIZE

RULES = {"floor": _native.MX_FLOOR, "up": _native.MX_UP}
_DTYPES = {torch.bfloat16: _native.T_BF16, torch.float16: _native.T_FP16,
           torch.float32: _native.T_FP32}
_current_device = torch._C._cuda_getDevice
_raw_stream = torch._C._cuda_getCurrentRawStream


def _code_bytes(rows: int, cols: int) -> int:
    return rows * ((cols + MX_GROUP_SIZE - 1) // MX_GROUP_SIZE) * (MX_GROUP_SIZE // 2)


def _packed_bytes(rows: int, cols: int) -> int:
    """Bytes of the packed scales of [rows][cols]: rows to 256, groups to 8."""
    return (rows + 255) // 256 * 256 * ((cols + 255) // 256 * 8)


@functools.lru_cache(maxsize=4096)
def _places(rows: int, cols: int) -> tuple[int, int]:
    """Where the scales begin behind the codes, and where they end (multiples of 256)."""
    scales = (_code_bytes(rows, cols) + 255) // 256 * 256
    return scales, scales + _packed_bytes(rows, cols)


class MxTensor:
    """A [rows][cols] MX FP4 matrix.

    ``codes`` is uint8 [rows][ceil(cols / 32) * 16] (two codes a byte, zeros past
    cols), ``scales`` the E8M0 scales in the layout of ``tcb_mx_scales_pack``.
    """

    __slots__ = ("rows", "cols", "index", "codes_ptr", "scales_ptr", "_held")

    def __init__(self, codes: torch.Tensor, scales: torch.Tensor, rows: int, cols: int):
        if codes.dtype != torch.uint8 or scales.dtype != torch.uint8:
            raise TypeError("MX codes and scales are uint8")
        if codes.shape != (rows, (cols + 31) // 32 * 16):
            raise ValueError(f"codes of a {rows} x {cols} MX tensor are "
                             f"[{rows}][{(cols + 31) // 32 * 16}], got {list(codes.shape)}")
        if scales.numel() != _packed_bytes(rows, cols):
            raise ValueError(f"packed scales of a {rows} x {cols} MX tensor are "
                             f"{_packed_bytes(rows, cols)} bytes, got {scales.numel()}")
        if not (codes.is_contiguous() and scales.is_contiguous()):
            raise ValueError("MX codes and scales are contiguous")
        index = codes.get_device()
        if index < 0 or index != scales.get_device():
            raise ValueError("MX codes and scales are on one CUDA device")
        self.rows, self.cols, self.index = rows, cols, index
        self.codes_ptr, self.scales_ptr = codes.data_ptr(), scales.data_ptr()
        self._held = (codes, scales)

    @classmethod
    def empty_on(cls, other: torch.Tensor, rows: int, cols: int) -> "MxTensor":
        """Uninitialised, codes and scales in one allocation on another tensor's device."""
        offset, size = _places(rows, cols)
        held = other.new_empty(size, dtype=torch.uint8)
        t = cls.__new__(cls)
        t.rows, t.cols, t.index, t._held = rows, cols, held.get_device(), held
        t.codes_ptr = start = held.data_ptr()
        t.scales_ptr = start + offset
        return t

    @classmethod
    def two_on(cls, other: torch.Tensor, first: tuple[int, int],
               second: tuple[int, int]) -> "tuple[MxTensor, MxTensor]":
        """Two in one allocation, which lives as long as either (an allocation takes
        the host 1.7 us)."""
        a, b = cls.__new__(cls), cls.__new__(cls)
        offset, size = _places(*first)
        offset_b, size_b = _places(*second)
        held = other.new_empty(size + size_b, dtype=torch.uint8)
        a.rows, a.cols = first
        b.rows, b.cols = second
        a._held = b._held = held
        a.index = b.index = held.get_device()
        a.codes_ptr = start = held.data_ptr()
        a.scales_ptr = start + offset
        b.codes_ptr = start + size
        b.scales_ptr = start + size + offset_b
        return a, b

    @classmethod
    def from_rows(cls, codes: torch.Tensor, scales: torch.Tensor, cols: int) -> "MxTensor":
        """From codes and plain E8M0 scales [rows][ceil(cols / 32)], which are packed here."""
        rows, groups = codes.shape[0], (cols + 31) // 32
        if scales.dtype != torch.uint8 or scales.shape != (rows, groups) or \
                not scales.is_contiguous() or not scales.is_cuda:
            raise ValueError(f"plain scales are contiguous uint8 [{rows}][{groups}] on a CUDA device")
        packed = torch.empty(_packed_bytes(rows, cols), dtype=torch.uint8, device=scales.device)
        if packed.numel():
            with torch.cuda.device(scales.device):
                _native.mx_scales_pack(scales, packed, rows, groups)
        return cls(codes, packed, rows, cols)

    @property
    def shape(self) -> tuple[int, int]:
        return self.rows, self.cols

    @property
    def device(self) -> torch.device:
        return torch.device("cuda", self.index)

    def _any(self) -> torch.Tensor:
        return self._held[0] if isinstance(self._held, tuple) else self._held

    def _part(self, address: int, size: int) -> torch.Tensor:
        return self._held.narrow(0, address - self._held.data_ptr(), size)

    @property
    def codes(self) -> torch.Tensor:
        if isinstance(self._held, tuple):
            return self._held[0]
        return self._part(self.codes_ptr, _code_bytes(self.rows, self.cols)).view(
            self.rows, (self.cols + 31) // 32 * 16)

    @property
    def scales(self) -> torch.Tensor:
        if isinstance(self._held, tuple):
            return self._held[1]
        return self._part(self.scales_ptr, _packed_bytes(self.rows, self.cols))

    def __repr__(self) -> str:
        return f"MxTensor({self.rows} x {self.cols}, {self.device})"


def _call(name: str, index: int, *args) -> None:
    """The library's entry point on the current stream of device `index`, with it current."""
    fn = getattr(_native.calls(), name)
    if index == _current_device():
        status = fn(*args, _raw_stream(index))
    else:
        with torch.cuda.device(index):
            status = fn(*args, _raw_stream(index))
    if status:
        raise _native.TcbError(status, name)


def _dtype_code(dtype: torch.dtype, what: str) -> int:
    code = _DTYPES.get(dtype)
    if code is None:
        raise TypeError(f"{what} is bf16, fp16 or fp32, got {dtype}")
    return code


def _matrix(x: torch.Tensor, what: str) -> torch.Tensor:
    """x [..., cols] as a matrix [rows][cols] of the same memory."""
    if x.dim() == 0:
        raise ValueError(f"{what} has at least one axis")
    if x.dim() == 1:
        return x.unsqueeze(0)
    rows = 1
    for n in x.shape[:-1]:
        rows *= n
    try:
        return x.view(rows, x.shape[-1])
    except RuntimeError:
        raise ValueError(f"the leading axes of {what} do not merge into rows of one stride; "
                         "pass a contiguous tensor") from None


def _layout(x: torch.Tensor) -> tuple[int, int, int | None]:
    """Rows, columns and pitch (elements from one row to the next) of a matrix; no
    pitch where its rows are not contiguous or overlap."""
    rows, cols = x.shape
    down, along = x.stride()
    if along != 1 and cols > 1:
        return rows, cols, None
    if rows <= 1:
        return rows, cols, (cols + 7) // 8 * 8  # one row: any pitch does
    return rows, cols, down if down >= cols else None


def _device_index(x: torch.Tensor, what: str) -> int:
    index = x.get_device()
    if index < 0:
        raise ValueError(f"{what} is on a CUDA device")
    return index


def _quantizable(x: torch.Tensor, rule: str) -> torch.Tensor:
    """x as a matrix, once its type, its device and the rule are known to be quantize's."""
    _dtype_code(x.dtype, "x")
    if rule not in RULES:
        raise ValueError(f"rule is one of {sorted(RULES)}, got {rule!r}")
    _device_index(x, "x")
    return x if x.dim() == 2 else _matrix(x, "x")


def _quantize(x: torch.Tensor, rule: str, by_row: MxTensor | None, by_col: MxTensor | None) -> None:
    """The matrix x into by_row (as it is), by_col (transposed) or both."""
    r, c, pitch = _layout(x)
    if pitch is None:  # a transposed view: its rows are the columns of what lies in memory
        by_row, by_col = by_col, by_row
        r, c, pitch = _layout(x.t())
        if pitch is None:
            raise ValueError("one axis of x has to be contiguous and its rows must not overlap")
    if r and c:
        _call("tcb_mx_quantize", x.get_device(), _DTYPES[x.dtype], x.data_ptr(), r, c, pitch, RULES[rule],
              by_row and by_row.codes_ptr, by_row and by_row.scales_ptr,
              by_col and by_col.codes_ptr, by_col and by_col.scales_ptr)


def quantize(x: torch.Tensor, *, rule: str = "floor") -> MxTensor:
    """x [..., cols] as an MX tensor [rows][cols], groups of 32 along the last axis.

    ``rule="floor"`` is the OCP MX scale, 2^(floor(log2 max|v|) - 2): a largest value
    between 6 and 8 scales saturates at 6.  ``rule="up"`` takes the least power of
    two that holds the largest value.  Values are rounded to nearest even; a group
    with an infinity or a NaN becomes NaN as a whole.  A transposed view is read in
    place.
    """
    x = _quantizable(x, rule)
    rows = MxTensor.empty_on(x, *x.shape)
    _quantize(x, rule, rows, None)
    return rows


def quantize_pair(x: torch.Tensor, *, rule: str = "floor") -> tuple[MxTensor, MxTensor]:
    """quantize(x) and quantize(x^T) (x as a matrix [rows][cols]) in one read of x."""
    x = _quantizable(x, rule)
    r, c = x.shape
    rows, cols = MxTensor.empty_on(x, r, c), MxTensor.empty_on(x, c, r)  # either may outlive the other
    _quantize(x, rule, rows, cols)
    return rows, cols


def dequantize(q: MxTensor, dtype: torch.dtype = torch.bfloat16, *,
               out: torch.Tensor | None = None) -> torch.Tensor:
    """The values of q, rounded once to `dtype` (or to out's type)."""
    y, code, pitch = _output(out, q, q.rows, q.cols, dtype)
    if q.rows and q.cols:
        _call("tcb_mx_dequantize", q.index, code, q.codes_ptr, q.scales_ptr, q.rows, q.cols,
              y.data_ptr(), pitch)
    return y


def _output(out: torch.Tensor | None, q: MxTensor, rows: int, cols: int,
            dtype: torch.dtype) -> tuple[torch.Tensor, int, int]:
    """`out`, or a new tensor on q's device; the library's code of its type; its pitch."""
    if out is None:
        code = _dtype_code(dtype, "the output")
        return q._any().new_empty((rows, cols), dtype=dtype), code, cols
    code = _dtype_code(out.dtype, "out")
    if out.shape != (rows, cols):
        raise ValueError(f"out is [{rows}][{cols}], got {list(out.shape)}")
    if out.get_device() != q.index:
        raise ValueError(f"out is on {out.device}, the operands are on {q.device}")
    pitch = _layout(out)[2]
    if pitch is None:
        raise ValueError("the rows of out have to be contiguous and must not overlap")
    return out, code, pitch


def _bias(bias: torch.Tensor | None, n: int, y: torch.Tensor) -> int | None:
    """Address of a bias [n] of y's type."""
    if bias is None:
        return None
    if bias.dtype != y.dtype:
        raise TypeError(f"bias has the output's type {y.dtype}, got {bias.dtype}")
    if bias.shape != (n,) or (n > 1 and bias.stride(0) != 1):
        raise ValueError(f"bias is a contiguous [{n}], got {list(bias.shape)}")
    if bias.get_device() != y.get_device():
        raise ValueError(f"bias is on {bias.device}, the operands are on {y.device}")
    return bias.data_ptr()


def matmul(a: MxTensor, b: MxTensor, *, bias: torch.Tensor | None = None,
           dtype: torch.dtype = torch.bfloat16, out: torch.Tensor | None = None,
           status: torch.Tensor | None = None) -> torch.Tensor:
    """a [M][K] . b [N][K]^T (+ bias [N]) in `dtype` (or out's type).

    ``status`` (an int32 device word) receives an error of a device-side wait; without
    one such an error is not reported, and what the wait's tiles should have held is
    left unwritten.
    """
    m, n, k = a.rows, b.rows, a.cols
    if k != b.cols:
        raise ValueError(f"a has {k} columns and b {b.cols}")
    if a.index != b.index:
        raise ValueError(f"a is on {a.device} and b on {b.device}")
    if k == 0:
        raise ValueError("a product over no columns")
    y, code, pitch = _output(out, a, m, n, dtype)
    bias_ptr = _bias(bias, n, y)
    if m and n:
        _call("tcb_mx_gemm", a.index, a.codes_ptr, a.scales_ptr, b.codes_ptr, b.scales_ptr, bias_ptr,
              code, y.data_ptr(), pitch, m, n, k, _status(status, a.index))
    return y


def _status(status: torch.Tensor | None, index: int) -> int | None:
    """Address of a status word on device `index`."""
    if status is None:
        return None
    if status.dtype != torch.int32 or status.numel() < 1:
        raise TypeError(f"status is an int32 word, got {status.dtype} {list(status.shape)}")
    if status.get_device() != index:
        raise ValueError(f"status is on {status.device}, the operands are on cuda:{index}")
    return status.data_ptr()


# A size for a size: worked out by the library once per pair.
_workspace_bytes = functools.lru_cache(maxsize=1024)(_native.mx_linear_workspace_bytes)


def linear(x: torch.Tensor, w: MxTensor, *, bias: torch.Tensor | None = None,
           dtype: torch.dtype | None = None, out: torch.Tensor | None = None,
           status: torch.Tensor | None = None) -> torch.Tensor:
    """x [..., K] . w [N][K]^T (+ bias [N]) with bf16 or fp16 x, in `dtype` (default x's).

    Only the weight is rounded to MX FP4: x takes part as MX digits of three bits and
    fp32 products with what these leave, so small values count in full beside large
    ones.  Rows that leave much (a value 2^14 times the others, 2^11 in fp16, in every
    group of 32) take longer.  The first digit may be a seventh larger than its value, so
    sums that come within that of fp32's largest number may be infinite.  A few rows
    cost little more than reading w once, a prompt's several products of MX rows
    (quantise x too where that matters).  ``out`` is a matrix [rows][N]; ``status`` as in
    :func:`matmul`.
    """
    x_dtype = x.dtype
    if x_dtype != torch.bfloat16 and x_dtype != torch.float16:
        raise TypeError(f"x is bf16 or fp16, got {x_dtype}")
    if _device_index(x, "x") != w.index:
        raise ValueError(f"x is on {x.device} and w on {w.device}")
    flat = x if x.dim() == 2 else _matrix(x, "x")
    m, k, x_pitch = _layout(flat)
    n = w.rows
    if k != w.cols:
        raise ValueError(f"x has {k} columns and w {w.cols}")
    if k == 0:
        raise ValueError("a product over no columns")
    if x_pitch is None:
        raise ValueError("the rows of x have to be contiguous and must not overlap")
    y, code, pitch = _output(out, w, m, n, x_dtype if dtype is None else dtype)
    bias_ptr = _bias(bias, n, y)
    if m and n:
        need = _workspace_bytes(m, k)
        space = flat.new_empty(need, dtype=torch.uint8) if need else None
        _call("tcb_mx_linear", w.index, _DTYPES[x_dtype], flat.data_ptr(), x_pitch, w.codes_ptr,
              w.scales_ptr, bias_ptr, code, y.data_ptr(), pitch, m, n, k, _native._ptr(space), need,
              _status(status, w.index))
    return y if out is not None or flat is x else y.view(*x.shape[:-1], n)


@dataclass
class LinearSaved:
    """What linear_backward needs of the forward pass: x and w quantised along the
    axes that the gradients' products sum over, and the gradients' types."""

    x: MxTensor  # x^T [in][tokens]
    w: MxTensor  # w^T [in][out]
    x_shape: tuple
    x_dtype: torch.dtype
    w_dtype: torch.dtype
    rule: str


def linear_forward(x: torch.Tensor, w: torch.Tensor, *, rule: str = "floor",
                   status: torch.Tensor | None = None) -> tuple[torch.Tensor, LinearSaved]:
    """y = Q(x) . Q(w)^T for x [..., in], w [out][in], and what the backward pass needs.

    Each of x and w is read once and quantised along both axes.  ``status`` as in
    :func:`matmul`.
    """
    if w.dim() != 2 or x.dim() == 0 or x.shape[-1] != w.shape[1]:
        raise ValueError(f"x is [..., in] and w [out][in], got {list(x.shape)} and {list(w.shape)}")
    if x.get_device() != w.get_device():
        raise ValueError(f"x is on {x.device} and w on {w.device}")
    flat = _quantizable(x, rule)
    _quantizable(w, rule)
    tokens, inner = flat.shape
    outer = w.shape[0]
    x_rows, w_rows = MxTensor.two_on(w, (tokens, inner), (outer, inner))
    x_cols, w_cols = MxTensor.two_on(w, (inner, tokens), (inner, outer))
    _quantize(flat, rule, x_rows, x_cols)
    _quantize(w, rule, w_rows, w_cols)
    y = matmul(x_rows, w_rows, dtype=x.dtype, status=status)
    saved = LinearSaved(x_cols, w_cols, tuple(x.shape), x.dtype, w.dtype, rule)
    return y if x.dim() == 2 else y.view(*x.shape[:-1], w.shape[0]), saved


def linear_backward(dy: torch.Tensor, saved: LinearSaved, *, need_dx: bool = True, need_dw: bool = True,
                    status: torch.Tensor | None = None) -> tuple[torch.Tensor | None, torch.Tensor | None]:
    """(dx, dw) of y = Q(x) . Q(w)^T for the gradient dy [..., out] of y.

    dx = Q(dy) . Q(w^T)^T in x's type and shape, dw = Q(dy^T) . Q(x^T)^T in w's type
    (None where not needed); with no rows dw is zero, with no outputs dx.
    ``status`` as in :func:`matmul`, for both products.
    """
    out_features, in_features = saved.w.cols, saved.w.rows
    shape = saved.x_shape[:-1] + (out_features,)
    if tuple(dy.shape) != shape:
        raise ValueError(f"dy is {list(shape)}, got {list(dy.shape)}")
    if dy.get_device() != saved.x.index:
        raise ValueError(f"dy is on {dy.device}, the forward pass was on {saved.x.device}")
    dx = dw = dy_rows = dy_cols = None
    if need_dx or need_dw:
        flat = _quantizable(dy, saved.rule)
        tokens = flat.shape[0]
        if need_dx and need_dw:
            dy_rows, dy_cols = MxTensor.two_on(flat, (tokens, out_features), (out_features, tokens))
        elif need_dx:
            dy_rows = MxTensor.empty_on(flat, tokens, out_features)
        else:
            dy_cols = MxTensor.empty_on(flat, out_features, tokens)
        _quantize(flat, saved.rule, dy_rows, dy_cols)
    if need_dx:
        if out_features == 0:
            dx = torch.zeros(saved.x_shape, dtype=saved.x_dtype, device=dy.device)
        else:
            dx = matmul(dy_rows, saved.w, dtype=saved.x_dtype, status=status)
            if len(saved.x_shape) != 2:
                dx = dx.view(saved.x_shape)
    if need_dw:
        if saved.x.cols == 0:
            dw = torch.zeros((out_features, in_features), dtype=saved.w_dtype, device=dy.device)
        else:
            dw = matmul(dy_cols, saved.x, dtype=saved.w_dtype, status=status)
    return dx, dw
