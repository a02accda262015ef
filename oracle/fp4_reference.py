"""The microscaled 4-bit formats in 64 bits, on the CPU: what the kernels are held to.

Nothing here shares code with the kernels: numbers come from tables and nearest-value searches. The definition rounds a
few steps of the e4m3 format to f32 on purpose (minicompiler_b200_device.h says which); `f32` marks them.
"""

from __future__ import annotations

import numpy as np

BLOCK = {"e8m0_32": 32, "e4m3_16": 16}
MAGNITUDES = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])
# byte 0 .. 0x7E of e4m3 without a sign: 3 bits of mantissa, bias 7, no infinity; 0x7F is NaN
E4M3 = np.array([(b & 7) * 2.0 ** -9 if b < 8 else (1 + (b & 7) / 8.0) * 2.0 ** ((b >> 3) - 7) for b in range(0x7F)])


def f32(x):
    with np.errstate(over="ignore"):
        return np.asarray(x, dtype=np.float32).astype(np.float64)


def nearest_even(x, table):
    """Index of the nearest entry of an increasing table; of two equally near ones the even index. x >= 0; past the end: the last."""
    x = np.minimum(np.asarray(x, dtype=np.float64), table[-1])
    hi = np.clip(np.searchsorted(table, x, side="left"), 1, len(table) - 1)
    lo = hi - 1
    down, up = x - table[lo], table[hi] - x
    take_hi = (up < down) | ((up == down) & (hi % 2 == 0))
    return np.where(take_hi, hi, lo)


def tensor_scale(x):
    a = np.abs(np.asarray(x, dtype=np.float64))
    a = a[np.isfinite(a)]
    amax = a.max() if a.size else 0.0
    return 1.0 if amax == 0 else max(float(f32(amax / 2688.0)), 2.0 ** -120)


def quantize(x, fmt, g=1.0):
    """x [rows, cols], values of f32 or narrower -> (codes [rows, cols] 0..15, scale bytes [rows, blocks])."""
    x = np.asarray(x, dtype=np.float64)
    rows, cols = x.shape
    block = BLOCK[fmt]
    blocks = -(-cols // block)
    padded = np.zeros((rows, blocks * block))
    padded[:, :cols] = x
    padded = padded.reshape(rows, blocks, block)
    bad = ~np.isfinite(padded).all(axis=2)
    padded = np.where(bad[:, :, None], 0.0, padded)
    amax = np.abs(padded).max(axis=2)
    if fmt == "e8m0_32":
        e = np.frexp(amax)[1] - 1 - 2  # floor(log2 amax) - 2
        e = np.where(amax == 0, -127, np.maximum(e, -127))
        scale = np.where(bad, 255, e + 127)
        y = padded / np.exp2(e.astype(np.float64))[:, :, None]
    else:
        g = float(g)
        ok = np.isfinite(g) and g > 0
        bad = bad | (not ok)
        six_g = f32(6.0 * g) if ok else 1.0
        with np.errstate(over="ignore", divide="ignore", invalid="ignore"):
            t = f32(amax / six_g)
            scale = nearest_even(t, E4M3)
            step = f32(E4M3[scale] * (g if ok else 1.0))
            inverse = np.where(step == 0, 0.0, np.minimum(f32(1.0 / np.where(step == 0, 1.0, step)), float(np.finfo(np.float32).max)))
            y = f32(padded * inverse[:, :, None])
        scale = np.where(bad, 0x7F, scale)
    code = nearest_even(np.abs(y), MAGNITUDES) + 8 * np.signbit(y)
    code = np.where(bad[:, :, None], 0, code).reshape(rows, blocks * block)[:, :cols]
    return code.astype(np.uint8), scale.astype(np.uint8)


def code_pitch(cols):
    return -(-cols // 32) * 16


def pack(code, scale, fmt):
    """Numbers -> the two arrays in memory: codes [rows, pitch], scales [row tiles, k tiles, 512]."""
    rows, cols = code.shape
    full = np.zeros((rows, 2 * code_pitch(cols)), dtype=np.uint8)
    full[:, :cols] = code
    blocks = scale.shape[1]
    tiles = np.zeros((-(-rows // 128), -(-blocks // 4), 512), dtype=np.uint8)
    r, b = np.arange(rows)[:, None], np.arange(blocks)[None, :]
    tiles[r // 128, b // 4, r % 32 * 16 + r // 32 % 4 * 4 + b % 4] = scale
    return full[:, 0::2] | (full[:, 1::2] << 4), tiles


def values(code, scale, fmt, g=1.0):
    """The numbers that codes and scale bytes stand for, in 64 bits."""
    sign = np.where(code >= 8, -1.0, 1.0)
    if fmt == "e8m0_32":
        s = np.where(scale == 255, np.nan, np.exp2(scale.astype(np.float64) - 127.0))
    else:
        s = np.append(E4M3, np.nan)[scale] * float(g)
    return sign * MAGNITUDES[code & 7] * np.repeat(s, BLOCK[fmt], axis=1)[:, : code.shape[1]]
