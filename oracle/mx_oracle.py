"""MXFP4 quantization restated in numpy: E2M1 elements with one power of two
per 32 values, in the layouts the library writes.

The shared exponent of a block is floor(log2(amax)) - 2, at least -127 (-127
for a block of zeros); elements are the nearest E2M1 value of v / 2^e, ties to
the even code, at most 6 in magnitude.  A block that holds an infinity or a
NaN has scale code 0xFF.
"""
from __future__ import annotations

import numpy as np

from . import nvfp4_oracle as orc

GRID = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])


def encode(a):
    """E2M1 codes (0..7) of non-negative float64 values."""
    hi = np.minimum(np.searchsorted(GRID, a), 7)
    lo = np.maximum(hi - 1, 0)
    up, down = GRID[hi] - a, a - GRID[lo]
    return np.where((up < down) | ((up == down) & (hi % 2 == 0)), hi, lo).astype(np.uint8)


def quantize(v):
    """float array [rows, k], k % 32 == 0 -> (packed u8 [rows, k/2], swizzled scale bytes)."""
    v = np.asarray(v, dtype=np.float64)
    rows, k = v.shape
    b = v.reshape(rows, k // 32, 32)
    amax = np.abs(b).max(axis=2) if rows else np.zeros((0, k // 32))
    bad = ~np.isfinite(b).all(axis=2)
    with np.errstate(all="ignore"):
        _, ex = np.frexp(np.where(bad, 1.0, amax))
    e = np.where(amax > 0, np.maximum(ex.astype(np.int64) - 1 - 2, -127), -127)
    with np.errstate(all="ignore"):
        scaled = np.ldexp(np.where(np.isfinite(b), b, 0.0), -e[:, :, None].astype(np.int32))
    q = encode(np.abs(scaled)) | (np.signbit(b).astype(np.uint8) << 3)
    q = q.reshape(rows, k)
    packed = q[:, 0::2] | (q[:, 1::2] << 4)
    code = np.where(bad, 255, e + 127).astype(np.uint8)
    pr, pc = orc.mx_scale_shape(rows, k)
    s = np.zeros(pr * pc, dtype=np.uint8)
    rr, cc = np.meshgrid(np.arange(rows), np.arange(k // 32), indexing="ij")
    s[orc.swizzle_offset(rr, cc, pc)] = code
    return packed, s.reshape(pr, pc)


def quantize_t(v):
    """The transpose of float [rows, cols], rows filled up with zeros to a multiple of 32."""
    v = np.asarray(v, dtype=np.float64)
    full = np.zeros((-(-v.shape[0] // 32) * 32, v.shape[1]))
    full[:v.shape[0]] = v
    return quantize(np.ascontiguousarray(full.T))
