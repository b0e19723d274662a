"""Plain 64-bit implementations of the microscaled (MX) operators, in numpy: the definitions the tests hold the library to."""
from __future__ import annotations

import numpy as np

BLOCK = 32
LARGEST = {"mxf8": 448.0, "mxf4": 6.0}
U = 2.0 ** -24  # half a step of fp32, relative


def _grid(kind: str) -> np.ndarray:
    """The non-negative values of the element type, by code."""
    if kind == "mxf4":
        return np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6])
    e, m = np.divmod(np.arange(127), 8)
    return np.where(e == 0, m / 8 * 2.0 ** -6, (1 + m / 8) * 2.0 ** (e - 7.0))


def scale_codes(x: np.ndarray, kind: str) -> np.ndarray:
    """E8M0 code of every block: the least e >= -127 with amax <= LARGEST * 2^e; 255 for a block with an infinity or a NaN."""
    rows, O = x.shape
    out = np.zeros((rows, -(-O // BLOCK)), np.uint8)
    for b in range(out.shape[1]):
        block = np.abs(x[:, b * BLOCK:(b + 1) * BLOCK].astype(np.float64))
        for r in range(rows):
            amax = block[r].max()
            if not np.isfinite(amax):
                out[r, b] = 255
                continue
            e = -127
            if amax > 0:
                e = max(-127, int(np.floor(np.log2(amax))) - 12)
                while amax > LARGEST[kind] * 2.0 ** e:
                    e += 1
            out[r, b] = e + 127
    return out


def quantize(x: np.ndarray, kind: str):
    """(element codes uint8 [rows, O], scale codes): nearest element, ties to the even code."""
    x = x.astype(np.float64)
    codes = scale_codes(x, kind)
    full = np.repeat(codes, BLOCK, 1)[:, :x.shape[1]].astype(int)
    t = np.where(full == 255, 0.0, x) * 2.0 ** (127.0 - np.where(full == 255, 127, full))
    grid = _grid(kind)
    a = np.abs(t)
    hi = np.clip(np.searchsorted(grid, a), 1, len(grid) - 1)
    lo = hi - 1
    dlo, dhi = a - grid[lo], grid[hi] - a
    c = np.where((dlo < dhi) | ((dlo == dhi) & (lo % 2 == 0)), lo, hi)
    sign = 0x80 if kind == "mxf8" else 8
    return (c | np.where(np.signbit(t) & (full != 255), sign, 0)).astype(np.uint8), codes


def element_values(codes: np.ndarray, kind: str) -> np.ndarray:
    sign, most = (0x80, 127) if kind == "mxf8" else (8, 8)
    grid = np.append(_grid(kind), np.nan) if kind == "mxf8" else _grid(kind)
    return np.where(codes & sign, -1.0, 1.0) * grid[codes & (most if kind == "mxf8" else 7)]


def values(codes: np.ndarray, scales: np.ndarray, kind: str) -> np.ndarray:
    s = np.repeat(scales, BLOCK, 1)[:, :codes.shape[1]].astype(np.float64)
    return element_values(codes, kind) * np.where(s == 255, np.nan, 2.0 ** (s - 127))


def pack(codes: np.ndarray) -> np.ndarray:
    if codes.shape[1] % 2:
        codes = np.pad(codes, ((0, 0), (0, 1)))
    return codes[:, 0::2] | (codes[:, 1::2] << 4)


def unpack(data: np.ndarray, O: int) -> np.ndarray:
    return np.stack([data & 15, data >> 4], -1).reshape(data.shape[0], -1)[:, :O]


def product(row_ptr, col, val, B):
    """(C, sum of |a b|, entries of the longest row), in 64 bits; rows without entries are 0."""
    M = len(row_ptr) - 1
    C, absC = np.zeros((M, B.shape[1])), np.zeros((M, B.shape[1]))
    for r in range(M):
        p = slice(row_ptr[r], row_ptr[r + 1])
        t = val[p].astype(np.float64)[:, None] * B[col[p]]
        C[r], absC[r] = t.sum(0), np.abs(t).sum(0)
    return C, absC, int(np.diff(row_ptr).max(initial=0))


def norm(s: np.ndarray, w: np.ndarray, eps: float):
    """(y, inv_rms) of the stored sum s."""
    s = s.astype(np.float64)
    inv = 1 / np.sqrt((s * s).mean(1) + eps)
    return s * inv[:, None] * w.astype(np.float64), inv


def norm_backward(dy, w, s, inv, d_residual):
    """(dx, dweight, bound of |dx|'s terms, sum of |dw|'s terms)."""
    dy, w, s, inv = (np.asarray(t, np.float64) for t in (dy, w, s, inv))
    inv = inv[:, None]
    g, O = dy * w, dy.shape[1]
    dr = 0.0 if d_residual is None else np.asarray(d_residual, np.float64)
    dx = dr + inv * g - s * inv ** 3 * (g * s).sum(1, keepdims=True) / O
    size = np.abs(dr) + np.abs(inv * g) + np.abs(s) * inv ** 3 * np.abs(g * s).sum(1, keepdims=True) / O
    t = dy * s * inv
    return dx, t.sum(0), size, np.abs(t).sum(0)
