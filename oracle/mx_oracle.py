"""Microscaled formats and products in numpy, from their definitions, in 64 bits.

value = code * scale * tensor scale g, one scale per block of a row:
    mxfp4  codes E2M1, blocks of 32, scales 2^e with e = max(floor(log2 max|x|) - 2, -127)
    nvfp4  codes E2M1, blocks of 16, scales E4M3 nearest to max|x| / (6 g)
    mxfp8  codes E4M3, blocks of 32, scales 2^e with e = max(floor(log2 max|x|) - 8, -127)
Codes are nearest (ties to the even code) to x / (scale g), at most the largest.
A block with a non-finite value has the scale NaN and zero codes.
"""

from __future__ import annotations

import numpy as np

BLOCK = {"mxfp4": 32, "nvfp4": 16, "mxfp8": 32}
EMAX = {"mxfp4": 2, "mxfp8": 8}
E2M1 = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6], np.float64)
# E4M3: 4 exponent bits (bias 7), 3 digits, subnormals below 2^-6; 0x7F is NaN
E4M3 = np.array([(m / 8 * 2.0**-6 if e == 0 else (1 + m / 8) * 2.0 ** (e - 7)) for e in range(16) for m in range(8)][:127],
                np.float64)


def nearest_code(v, table):
    """Index of the nearest magnitude of `table`, ties to the even index."""
    a = np.abs(v)
    middle = (table[1:] + table[:-1]) / 2
    low = np.searchsorted(middle, a, side="left")  # a == middle[i] -> i
    tie = (low < middle.size) & (a == middle[np.minimum(low, middle.size - 1)])
    return (low + (tie & (low % 2 == 1))).astype(np.uint8)


def quantise(x, fmt, g=1.0):
    """x [rows, cols] -> codes uint8 [rows, padded cols] (sign and magnitude, one
    a byte), scales uint8 [rows, blocks of the padded columns]."""
    x = np.asarray(x, np.float64)
    rows, cols = x.shape
    padded = -(-cols // 32) * 32
    b = np.zeros((rows, padded))
    b[:, :cols] = x
    b = b.reshape(rows, padded // BLOCK[fmt], BLOCK[fmt])
    finite = np.isfinite(b).all(2)
    b = np.where(finite[..., None], b, 0.0)
    a = np.abs(b).max(2)
    if fmt == "nvfp4":
        scales = nearest_code(a / (6.0 * g), E4M3)
        s = E4M3[scales] * g
        v = np.divide(b, s[..., None], out=np.zeros_like(b), where=s[..., None] > 0)
    else:
        e = np.where(a > 0, np.frexp(a)[1] - 1 - EMAX[fmt], -127)
        e = np.maximum(e, -127)
        scales = (e + 127).astype(np.uint8)
        v = b / np.exp2(e.astype(np.float64))[..., None]
    if fmt == "mxfp8":
        codes = nearest_code(v, E4M3) | (np.signbit(b).astype(np.uint8) << 7)
    else:
        codes = nearest_code(v, E2M1) | (np.signbit(b).astype(np.uint8) << 3)
    codes = np.where(finite[..., None], codes, 0).astype(np.uint8)
    scales = np.where(finite, scales, 0x7F if fmt == "nvfp4" else 0xFF).astype(np.uint8)
    return codes.reshape(rows, padded), scales


def values(codes, scales, fmt, g=1.0, cols=None):
    """What codes and scales stand for, float64 [rows, cols]."""
    table = E4M3 if fmt == "mxfp8" else E2M1
    sign = 7 if fmt == "mxfp8" else 3
    v = table[codes & ((1 << sign) - 1)] * np.where(codes >> sign & 1, -1.0, 1.0)
    if fmt == "nvfp4":
        s = np.append(E4M3, np.nan)[scales] * g
    else:
        s = np.where(scales == 255, np.nan, np.exp2(scales.astype(np.float64) - 127))
    v = v.reshape(v.shape[0], scales.shape[1], BLOCK[fmt]) * s[..., None]
    return v.reshape(v.shape[0], codes.shape[1])[:, :cols]


def held(x, fmt, g=1.0):
    """What x stands for after quantising."""
    return values(*quantise(x, fmt, g), fmt, g, np.asarray(x).shape[1])


def pack(codes, fmt):
    """Codes as the rows of a quantised matrix hold them."""
    return codes if fmt == "mxfp8" else codes[:, 0::2] | (codes[:, 1::2] << 4)


def tile_scales(scales):
    """Row-major scales [rows, blocks] in tiles of 128 rows x 4, 512 bytes each
    (missing rows and columns are 0)."""
    rows, blocks = scales.shape
    bands, tiles = -(-rows // 128), -(-blocks // 4)
    out = np.zeros((bands, tiles, 512), np.uint8)
    r, c = np.meshgrid(np.arange(rows), np.arange(blocks), indexing="ij")
    out[r // 128, c // 4, r % 32 * 16 + r // 32 % 4 * 4 + c % 4] = scales
    return out


def cache_slots(pages, page_rows, offsets, starts, rows):
    """Cache row of each packed row, -1 where it has none."""
    out = np.full(rows, -1, np.int64)
    for s in range(len(offsets) - 1):
        for t in range(max(0, offsets[s]), min(rows, offsets[s + 1])):
            position = (starts[s] if starts is not None else 0) + t - offsets[s]
            if 0 <= position < pages.shape[1] * page_rows and pages[s, position // page_rows] >= 0:
                out[t] = int(pages[s, position // page_rows]) * page_rows + position % page_rows
    return out


def linear(x, w, fmt, gx=1.0, gw=1.0, bias=None, slope=1.0, residual=None):
    """(y, sum of the products' magnitudes): y = leaky(x w^T + bias) + residual
    on what x and w stand for."""
    a, b = held(x, fmt, gx), held(w, fmt, gw)
    v = a @ b.T
    size = np.abs(a) @ np.abs(b).T
    if bias is not None:
        v = v + bias
        size = size + np.abs(bias)
    v = np.where(v >= 0, v, v * slope)
    if residual is not None:
        v = v + residual
        size = size + np.abs(residual)
    return v, size
