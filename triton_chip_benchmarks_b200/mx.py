"""Microscaled 4-bit floating point (MX FP4) on torch tensors.

An :class:`MxTensor` stands for a matrix whose values are E2M1 codes times a power
of two shared by 32 neighbours of a row (OCP MX).  The operators run on the
tensors' device and on its current stream, allocate their outputs through torch unless
``out`` is given, never synchronise, and can be captured into a CUDA graph:

* :func:`quantize`, :func:`quantize_pair`, :func:`dequantize`: between torch tensors
  (bf16, fp16, fp32) and MX tensors, along one axis or both in one read;
* :func:`matmul`: ``a . b^T`` of two MX tensors;
* :func:`linear`: 16-bit rows times an MX weight, for few rows (decoding);
* :func:`linear_forward`, :func:`linear_backward`: a linear layer's training step in
  MX products (both passes quantise their operands along the axis that the
  product sums over; gradients pass the rounding unchanged).

Results are rounded once, from fp32 sums.  Arguments that an operator does not take
raise ``TypeError`` (types) or ``ValueError`` (shapes, strides, devices); what the
library itself refuses raises :class:`_native.TcbError`.
"""

from __future__ import annotations

from dataclasses import dataclass

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


class MxTensor:
    """A [rows][cols] MX FP4 matrix.

    ``codes`` is uint8 [rows][ceil(cols / 32) * 16] (two codes a byte, zeros past
    cols), ``scales`` the E8M0 scales in the layout of ``tcb_mx_scales_pack``.
    """

    __slots__ = ("rows", "cols", "device", "codes_ptr", "scales_ptr", "_held")

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
        device = codes.device
        if device != scales.device or not codes.is_cuda:
            raise ValueError("MX codes and scales are on one CUDA device")
        self.rows, self.cols, self.device = rows, cols, device
        self.codes_ptr, self.scales_ptr = codes.data_ptr(), scales.data_ptr()
        self._held = (codes, scales)

    @classmethod
    def empty(cls, rows: int, cols: int, device: torch.device) -> "MxTensor":
        """Uninitialised, codes and scales in one allocation."""
        t = cls.__new__(cls)
        offset = (_code_bytes(rows, cols) + 255) // 256 * 256
        held = torch.empty(offset + _packed_bytes(rows, cols), dtype=torch.uint8, device=device)
        t.rows, t.cols, t.device, t._held = rows, cols, held.device, held
        t.codes_ptr = held.data_ptr()
        t.scales_ptr = t.codes_ptr + offset
        return t

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
    def codes(self) -> torch.Tensor:
        if isinstance(self._held, tuple):
            return self._held[0]
        return self._held[:_code_bytes(self.rows, self.cols)].view(self.rows, (self.cols + 31) // 32 * 16)

    @property
    def scales(self) -> torch.Tensor:
        if isinstance(self._held, tuple):
            return self._held[1]
        return self._held[self.scales_ptr - self.codes_ptr:]

    def __repr__(self) -> str:
        return f"MxTensor({self.rows} x {self.cols}, {self.device})"


def _call(name: str, device: torch.device, *args) -> None:
    """The library's entry point on the device's current stream, with the device current."""
    index = device.index
    fn = getattr(_native.load(), name)
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


def _rule_code(rule: str) -> int:
    if rule not in RULES:
        raise ValueError(f"rule is one of {sorted(RULES)}, got {rule!r}")
    return RULES[rule]


def _matrix(x: torch.Tensor, what: str) -> torch.Tensor:
    """x [..., cols] as a matrix [rows][cols] of the same memory."""
    if not x.is_cuda:
        raise ValueError(f"{what} is on a CUDA device")
    if x.dim() == 2:
        return x
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


def _pitch(x: torch.Tensor) -> int | None:
    """Elements from one row of a matrix to the next; None where its rows are not
    contiguous or overlap."""
    rows, cols = x.shape
    if cols > 1 and x.stride(1) != 1:
        return None
    if rows <= 1:
        return (cols + 7) // 8 * 8  # one row: any pitch does
    return x.stride(0) if x.stride(0) >= cols else None


def _quantize(x: torch.Tensor, rule: str, rows: bool, cols: bool):
    dtype = _dtype_code(x.dtype, "x")
    code = _rule_code(rule)
    x = _matrix(x, "x")
    pitch = _pitch(x)
    swap = pitch is None
    if swap:  # a transposed view: its rows are the columns of what lies in memory
        x = x.t()
        rows, cols = cols, rows
        pitch = _pitch(x)
        if pitch is None:
            raise ValueError("one axis of x has to be contiguous and its rows must not overlap")
    r, c = x.shape
    device = x.device
    by_row = MxTensor.empty(r, c, device) if rows else None
    by_col = MxTensor.empty(c, r, device) if cols else None
    if r and c:
        _call("tcb_mx_quantize", device, dtype, x.data_ptr(), r, c, pitch, code,
              by_row.codes_ptr if rows else None, by_row.scales_ptr if rows else None,
              by_col.codes_ptr if cols else None, by_col.scales_ptr if cols else None)
    return (by_col, by_row) if swap else (by_row, by_col)


def quantize(x: torch.Tensor, *, rule: str = "floor") -> MxTensor:
    """x [..., cols] as an MX tensor [rows][cols], groups of 32 along the last axis.

    ``rule="floor"`` is the OCP MX scale, 2^(floor(log2 max|v|) - 2): a largest value
    between 6 and 8 scales saturates at 6.  ``rule="up"`` takes the least power of
    two that holds the largest value.  Values are rounded to nearest even; a group
    with an infinity or a NaN becomes NaN as a whole.  A transposed view is read in
    place.
    """
    return _quantize(x, rule, True, False)[0]


def quantize_pair(x: torch.Tensor, *, rule: str = "floor") -> tuple[MxTensor, MxTensor]:
    """quantize(x) and quantize(x^T) (x as a matrix [rows][cols]) in one read of x."""
    return _quantize(x, rule, True, True)


def dequantize(q: MxTensor, dtype: torch.dtype = torch.bfloat16, *, out: torch.Tensor | None = None) -> torch.Tensor:
    """The values of q, rounded once to `dtype` (or to out's type)."""
    y = _output(out, q.device, q.rows, q.cols, dtype)
    if q.rows and q.cols:
        _call("tcb_mx_dequantize", q.device, _DTYPES[y.dtype], q.codes_ptr, q.scales_ptr, q.rows,
              q.cols, y.data_ptr(), _pitch(y))
    return y


def _output(out: torch.Tensor | None, device: torch.device, rows: int, cols: int,
            dtype: torch.dtype) -> torch.Tensor:
    if out is None:
        _dtype_code(dtype, "the output")
        return torch.empty((rows, cols), dtype=dtype, device=device)
    _dtype_code(out.dtype, "out")
    if out.shape != (rows, cols):
        raise ValueError(f"out is [{rows}][{cols}], got {list(out.shape)}")
    if out.device != device:
        raise ValueError(f"out is on {out.device}, the operands are on {device}")
    if _pitch(out) is None:
        raise ValueError("the rows of out have to be contiguous and must not overlap")
    return out


def _bias(bias: torch.Tensor | None, n: int, y: torch.Tensor) -> int | None:
    """Address of a bias [n] of y's type."""
    if bias is None:
        return None
    if bias.dtype != y.dtype:
        raise TypeError(f"bias has the output's type {y.dtype}, got {bias.dtype}")
    if bias.shape != (n,) or (n > 1 and bias.stride(0) != 1):
        raise ValueError(f"bias is a contiguous [{n}], got {list(bias.shape)}")
    if bias.device != y.device:
        raise ValueError(f"bias is on {bias.device}, the operands are on {y.device}")
    return bias.data_ptr()


def matmul(a: MxTensor, b: MxTensor, *, bias: torch.Tensor | None = None,
           dtype: torch.dtype = torch.bfloat16, out: torch.Tensor | None = None, status=None) -> torch.Tensor:
    """a [M][K] . b [N][K]^T (+ bias [N]) in `dtype` (or out's type).

    ``status`` (an int32 device word) receives an error of a device-side wait.
    """
    if a.cols != b.cols:
        raise ValueError(f"a has {a.cols} columns and b {b.cols}")
    if a.device != b.device:
        raise ValueError(f"a is on {a.device} and b on {b.device}")
    if a.cols == 0:
        raise ValueError("a product over no columns")
    y = _output(out, a.device, a.rows, b.rows, dtype)
    bias_ptr = _bias(bias, b.rows, y)
    if a.rows and b.rows:
        _call("tcb_mx_gemm", a.device, a.codes_ptr, a.scales_ptr, b.codes_ptr, b.scales_ptr, bias_ptr,
              _DTYPES[y.dtype], y.data_ptr(), _pitch(y), a.rows, b.rows, a.cols, _native._ptr(status))
    return y


def linear(x: torch.Tensor, w: MxTensor, *, bias: torch.Tensor | None = None,
           dtype: torch.dtype | None = None, out: torch.Tensor | None = None, status=None) -> torch.Tensor:
    """x [..., K] . w [N][K]^T (+ bias [N]) with bf16 or fp16 x, in `dtype` (default x's).

    Only the weight is rounded to MX FP4.  Meant for few rows: w is read once per 16
    rows of x (for many rows quantise x too and take :func:`matmul`).  ``out`` is a
    matrix [rows][N].
    """
    if x.dtype not in (torch.bfloat16, torch.float16):
        raise TypeError(f"x is bf16 or fp16, got {x.dtype}")
    lead = x.shape[:-1]
    m = _matrix(x, "x")
    if m.shape[1] != w.cols:
        raise ValueError(f"x has {m.shape[1]} columns and w {w.cols}")
    if m.device != w.device:
        raise ValueError(f"x is on {m.device} and w on {w.device}")
    if w.cols == 0:
        raise ValueError("a product over no columns")
    pitch = _pitch(m)
    if pitch is None:
        raise ValueError("the rows of x have to be contiguous and must not overlap")
    y = _output(out, m.device, m.shape[0], w.rows, x.dtype if dtype is None else dtype)
    bias_ptr = _bias(bias, w.rows, y)
    if m.shape[0] and w.rows:
        need = _native.mx_linear_workspace_bytes(m.shape[0], w.cols)
        space = torch.empty(need, dtype=torch.uint8, device=m.device) if need else None
        _call("tcb_mx_linear", m.device, _DTYPES[x.dtype], m.data_ptr(), pitch, w.codes_ptr,
              w.scales_ptr, bias_ptr, _DTYPES[y.dtype], y.data_ptr(), _pitch(y), m.shape[0], w.rows,
              w.cols, _native._ptr(space), need, _native._ptr(status))
    return y if out is not None or len(lead) == 1 else y.view(*lead, w.rows)


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


def linear_forward(x: torch.Tensor, w: torch.Tensor, *,
                   rule: str = "floor") -> tuple[torch.Tensor, LinearSaved]:
    """y = Q(x) . Q(w)^T for x [..., in], w [out][in], and what the backward pass needs.

    Each of x and w is read once and quantised along both axes.
    """
    if w.dim() != 2 or x.dim() == 0 or x.shape[-1] != w.shape[1]:
        raise ValueError(f"x is [..., in] and w [out][in], got {list(x.shape)} and {list(w.shape)}")
    if x.device != w.device:
        raise ValueError(f"x is on {x.device} and w on {w.device}")
    x_rows, x_cols = quantize_pair(x, rule=rule)
    w_rows, w_cols = quantize_pair(w, rule=rule)
    y = matmul(x_rows, w_rows, dtype=x.dtype)
    saved = LinearSaved(x_cols, w_cols, tuple(x.shape), x.dtype, w.dtype, rule)
    return y.view(*x.shape[:-1], w.shape[0]), saved


def linear_backward(dy: torch.Tensor, saved: LinearSaved, *, need_dx: bool = True,
                    need_dw: bool = True) -> tuple[torch.Tensor | None, torch.Tensor | None]:
    """(dx, dw) of y = Q(x) . Q(w)^T for the gradient dy [..., out] of y.

    dx = Q(dy) . Q(w^T)^T in x's type and shape, dw = Q(dy^T) . Q(x^T)^T in w's type
    (None where not needed); with no rows dw is zero.
    """
    out_features, in_features = saved.w.cols, saved.w.rows
    shape = saved.x_shape[:-1] + (out_features,)
    if tuple(dy.shape) != shape:
        raise ValueError(f"dy is {list(shape)}, got {list(dy.shape)}")
    if dy.device != saved.x.device:
        raise ValueError(f"dy is on {dy.device}, the forward pass was on {saved.x.device}")
    dy_rows, dy_cols = _quantize(dy, saved.rule, need_dx, need_dw) \
        if need_dx or need_dw else (None, None)
    dx = dw = None
    if need_dx:
        dx = matmul(dy_rows, saved.w, dtype=saved.x_dtype).view(saved.x_shape)
    if need_dw:
        if saved.x.cols == 0:
            dw = torch.zeros((out_features, in_features), dtype=saved.w_dtype, device=dy.device)
        else:
            dw = matmul(dy_cols, saved.x, dtype=saved.w_dtype)
    return dx, dw
