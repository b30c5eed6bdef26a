"""MX FP4 oracle (numpy, 64 bits) - test infrastructure.

The definition of the microscaled 4-bit operators from the OCP MX format: a group of
32 values shares the scale 2^e, e = floor(log2 max|v|) - 2 ("floor") or the least e
with 6 * 2^e >= max|v| ("up"), at least -127; each value becomes the nearest E2M1
code of v / 2^e, ties to the even code, saturating at 6.  A group of zeros has the
scale code 127, a group with an infinity or a NaN the code 255 and zero codes.
"""

from __future__ import annotations

import numpy as np

from .tensor import E2M1_VALUES, decode_e2m1, pack_e2m1_pairs

GROUP = 32
_GRID = np.array(E2M1_VALUES[:8])
_MIDDLE = (_GRID[1:] + _GRID[:-1]) / 2


def quantize(x: np.ndarray, rule: str) -> tuple[np.ndarray, np.ndarray]:
    """(packed codes [rows][groups * 16], scale codes [rows][groups]) of float64 x."""
    rows, cols = x.shape
    groups = -(-cols // GROUP)
    v = np.zeros((rows, groups * GROUP))
    v[:, :cols] = x
    v = v.reshape(rows, groups, GROUP)
    bad = ~np.isfinite(v).all(-1)
    top = np.where(np.isfinite(v), np.abs(v), 0.0).max(-1)
    _, exponent = np.frexp(top)  # top in [2^(exponent-1), 2^exponent)
    e = exponent.astype(np.int64) - 3
    if rule == "up":
        e += top > 6 * np.ldexp(1.0, e)
    e = np.maximum(e, -127)
    scaled = np.abs(v) / np.ldexp(1.0, e)[..., None]
    scaled = np.where(bad[..., None], 0.0, scaled)
    low = np.searchsorted(_MIDDLE, scaled, side="left")
    high = np.searchsorted(_MIDDLE, scaled, side="right")
    code = np.where((low != high) & (low % 2 == 1), high, low)  # a tie: the even one
    code = code + 8 * np.signbit(v)
    code = np.where(bad[..., None], 0, code).reshape(rows, -1).astype(np.uint8)
    scale = np.where(bad, 255, np.where(top == 0, 127, e + 127)).astype(np.uint8)
    return pack_e2m1_pairs(code), scale


def dequantize(codes: np.ndarray, scales: np.ndarray, cols: int) -> np.ndarray:
    """float64 values [rows][cols] of packed codes and scale codes [rows][groups]."""
    factor = np.where(scales == 255, np.nan, np.ldexp(1.0, scales.astype(np.int64) - 127))
    v = decode_e2m1(codes).reshape(codes.shape[0], -1, GROUP) * factor[..., None]
    return v.reshape(codes.shape[0], -1)[:, :cols]


def unpack_scales(packed: np.ndarray, rows: int, groups: int) -> np.ndarray:
    """The padded [rows_p][groups_p] scale codes of the packed layout."""
    rows_p, groups_p = -(-rows // 256) * 256, -(-groups // 8) * 8
    s = packed.reshape(rows_p // 128, groups_p // 8, 2, 32, 4, 4)
    # axes now: row block, group block, half, lane, row quarter, group
    return s.transpose(0, 4, 3, 1, 2, 5).reshape(rows_p, groups_p)
