"""Block-scaled FP8 in numpy, 64 bits, straight from the definition.

A row's block of 128 columns has the scale byte e, the smallest e >= 1 with
amax <= 448 * 2^(e-127) (255 when the block holds an infinity or a NaN), and
codes = E4M3(y * 2^(127-e)), round to nearest even."""
from __future__ import annotations

import numpy as np

BLOCK = 128

# The 127 non-negative finite E4M3 values, code order.
_GRID = np.array([m * 2.0 ** -9 if e == 0 else (1 + m / 8) * 2.0 ** (e - 7)
                  for e in range(16) for m in range(8)][:127])


def scale_byte(amax) -> np.ndarray:
    """Scale bytes of block maxima (float64)."""
    amax = np.asarray(amax, np.float64)
    out = np.full(amax.shape, 255, np.int64)
    fine = np.isfinite(amax)
    e = np.ones(amax.shape, np.int64)
    for _ in range(256):                       # the smallest e that holds amax, by search
        low = fine & (amax > 448.0 * np.exp2(e - 127.0))
        if not low.any():
            break
        e[low] += 1
    out[fine] = e[fine]
    return out.astype(np.uint8)


def encode(v) -> np.ndarray:
    """E4M3 codes of |v| <= 448 (or NaN -> 0x7f)."""
    v = np.asarray(v, np.float64)
    a = np.abs(v)
    hi = np.clip(np.searchsorted(_GRID, a), 0, 126)
    lo = np.maximum(hi - 1, 0)
    dh, dl = _GRID[hi] - a, a - _GRID[lo]
    code = np.where((dl < dh) | ((dl == dh) & (lo % 2 == 0)), lo, hi)
    code = code | np.where(np.signbit(v), 0x80, 0)
    return np.where(np.isnan(v), 0x7f, code).astype(np.uint8)


def decode(codes) -> np.ndarray:
    codes = np.asarray(codes, np.uint8)
    mag = codes & 0x7f
    v = np.where(mag == 127, np.nan, _GRID[np.minimum(mag, 126)])
    return np.where(codes & 0x80, -v, v)


def _blocks(y):
    rows, cols = y.shape
    kb = -(-cols // BLOCK)
    p = np.zeros((rows, kb * BLOCK))
    p[:, :cols] = y
    return p.reshape(rows, kb, BLOCK)


def _codes(blocks, e, cols):
    with np.errstate(invalid="ignore"):
        z = blocks * np.exp2(127.0 - e)
        z = np.where(e == 255, np.nan, z)
    return encode(z).reshape(z.shape[0], -1)[:, :cols]


def quantize(y):
    """(codes [rows, cols], scale bytes [rows, blocks]) of y."""
    b = _blocks(np.asarray(y, np.float64))
    amax = np.abs(b).max(-1)
    amax = np.where(np.isnan(b).any(-1), np.nan, amax)
    e = scale_byte(amax)
    return _codes(b, e[..., None].astype(np.int64), np.shape(y)[1]), e


def quantize_weight(w):
    """As quantize with one scale for each 128 x 128 block."""
    w = np.asarray(w, np.float64)
    rows = w.shape[0]
    b = _blocks(w)
    amax = np.abs(b).max(-1)
    e = np.concatenate([np.repeat(scale_byte(amax[r:r + BLOCK].max(0))[None], min(BLOCK, rows - r), 0)
                        for r in range(0, rows, BLOCK)])
    return _codes(b, e[..., None].astype(np.int64), w.shape[1]), e


def lay_out(e) -> np.ndarray:
    """[rows, blocks] scale bytes -> flat 128x4 blocked order."""
    rows, kb = e.shape
    katoms = -(-kb // 4)
    flat = np.zeros(-(-rows // 128) * 128 * katoms * 4, np.uint8)
    for r in range(rows):
        for k in range(kb):
            flat[((r // 128) * katoms + k // 4) * 512 + (r % 32) * 16 + (r % 128) // 32 * 4 + k % 4] = e[r, k]
    return flat


def values(codes, e) -> np.ndarray:
    """The values that codes [rows, cols] and scale bytes [rows, blocks] stand for."""
    s = np.where(e == 255, np.nan, np.exp2(e.astype(np.float64) - 127.0))
    return decode(codes) * np.repeat(s, BLOCK, 1)[:, :codes.shape[1]]


def rms_norm(x, weight, eps, residual=None):
    """(y, h) with h = x + residual, y = h / sqrt(mean(h^2) + eps) * weight."""
    h = np.asarray(x, np.float64)
    if residual is not None:
        h = h + np.asarray(residual, np.float64)
    return h / np.sqrt(np.mean(h * h, -1, keepdims=True) + eps) * np.asarray(weight, np.float64), h


def swiglu(gate, up):
    with np.errstate(over="ignore"):
        return gate / (1 + np.exp(-gate)) * up
