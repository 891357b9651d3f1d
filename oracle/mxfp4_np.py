"""MXFP4 in numpy, from the format's definition -- TEST INFRASTRUCTURE ONLY.

Blocks of 32 values, one scale 2^(byte - 127) each (255: NaN), four-bit codes: sign bit and a magnitude 0..7 for
0, 0.5, 1, 1.5, 2, 3, 4, 6.  Everything is computed in float64, one step after the other.
"""
from __future__ import annotations

import numpy as np

POINTS = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])
VALUES = np.concatenate([POINTS, -POINTS])


def quantize(x: np.ndarray):
    """(codes [rows, blocks * 16] bytes, scale bytes [rows, blocks]) of a float array [rows, cols]."""
    x = np.asarray(x, dtype=np.float64)
    rows, cols = x.shape
    blocks = (cols + 31) // 32
    v = np.zeros((rows, blocks * 32))
    v[:, :cols] = x
    v = v.reshape(rows, blocks, 32)
    top = np.abs(v).max(axis=2)
    bad = ~np.isfinite(top)
    with np.errstate(all="ignore"):
        _m, e = np.frexp(np.where(bad | (top == 0), 1.0, top))
    e = np.clip(e - 3, -127, 127)                       # floor(log2(top)) - 2
    e = np.where(top == 0, -127, e)
    v = np.where(bad[..., None], 0.0, v)
    a = np.abs(v) / np.exp2(e)[..., None]
    gap = np.abs(a[..., None] - POINTS)
    near = gap == gap.min(axis=-1, keepdims=True)
    even = near & (np.arange(8) % 2 == 0)
    code = np.where(even.any(axis=-1), even.argmax(axis=-1), near.argmax(axis=-1))
    code = (code + 8 * np.signbit(v)).astype(np.uint8).reshape(rows, blocks * 16, 2)
    return code[..., 0] | (code[..., 1] << 4), np.where(bad, 255, e + 127).astype(np.uint8)


def tile_scales(scales: np.ndarray) -> np.ndarray:
    """[rows, blocks] scale bytes to tiles of 128 rows x 4 blocks, by the address of each byte."""
    rows, blocks = scales.shape
    quads = (blocks + 3) // 4
    out = np.zeros((rows + 127) // 128 * quads * 512, np.uint8)
    r, b = np.arange(rows)[:, None], np.arange(blocks)[None, :]
    out[((r // 128) * quads + b // 4) * 512 + (r % 32) * 16 + (r % 128) // 32 * 4 + b % 4] = scales
    return out


def values(codes: np.ndarray, scales: np.ndarray) -> np.ndarray:
    """float64 values [rows, blocks * 32] of codes [rows, blocks * 16] and scale bytes [rows, blocks]."""
    rows, blocks = scales.shape
    v = np.empty((rows, blocks * 32))
    v[:, 0::2] = VALUES[codes & 15]
    v[:, 1::2] = VALUES[codes >> 4]
    s = np.where(scales == 255, np.nan, np.exp2(scales.astype(np.float64) - 127))
    return v * np.repeat(s, 32, axis=1)


def random_matrix(rows: int, blocks: int, rng, low: int = 118, high: int = 124):
    """Random codes and scale bytes in [low, high): (codes, scales, tiles, values)."""
    codes = rng.integers(0, 256, (rows, blocks * 16), dtype=np.uint8)
    scales = rng.integers(low, high, (rows, blocks), dtype=np.uint8)
    return codes, scales, tile_scales(scales), values(codes, scales)
