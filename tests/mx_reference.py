"""MXFP4 from its definition, in NumPy and 64 bits: what the tests hold the kernels to."""

import numpy as np

MAGNITUDES = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])
VALUES = np.concatenate([MAGNITUDES, -MAGNITUDES])


def ceil_div(a, b):
    return -(-a // b)


def quantize(x):
    """float [rows, cols] -> (codes [rows, cols], scales [rows, ceil(cols / 32)]), both uint8 and untiled."""
    x = np.asarray(x, dtype=np.float64)
    rows, cols = x.shape
    blocks = ceil_div(cols, 32)
    v = np.zeros((rows, blocks * 32))
    v[:, :cols] = x
    v = v.reshape(rows, blocks, 32)
    top = np.abs(v).max(axis=2)
    bad = ~np.isfinite(v).all(axis=2)
    exponent = np.frexp(np.where(bad | (top == 0), 1.0, top))[1] - 1          # floor(log2)
    scales = np.where(bad, 255, np.where(top == 0, 0, np.maximum(exponent - 2, -127) + 127))
    with np.errstate(invalid='ignore'):
        a = np.abs(v) * np.exp2(127.0 - scales)[:, :, None]
        # nearest magnitude; on a tie the even code
        distance = np.abs(np.minimum(a, 6.0)[..., None] - MAGNITUDES)
    first = distance.argmin(axis=-1)                                          # the lower of two that tie
    tie = distance[..., :-1] == distance[..., 1:]
    at = np.take_along_axis(tie, np.minimum(first, 6)[..., None], axis=-1)[..., 0] & (first < 7)
    code = np.where(at & (first % 2 == 1), first + 1, first)
    code = np.where(np.signbit(v), code | 8, code)
    code = np.where(bad[:, :, None], 0, code).reshape(rows, -1)[:, :cols]
    return code.astype(np.uint8), scales.astype(np.uint8)


def pack_codes(codes, pitch, fill=0):
    rows, cols = codes.shape
    out = np.full((rows, pitch // 2), fill, dtype=np.uint8)
    wide = np.zeros((rows, ceil_div(cols, 2) * 2), dtype=np.uint8)
    wide[:, :cols] = codes
    out[:, :wide.shape[1] // 2] = wide[:, 0::2] | (wide[:, 1::2] << 4)
    return out


def tile_scales(scales, cols, row_fill=0):
    """[rows, blocks] -> the tiled bytes; blocks beyond the row's end hold 0, rows beyond the last ``row_fill``."""
    rows, blocks = scales.shape
    across, groups = ceil_div(cols, 128), ceil_div(rows, 128)
    out = np.full((groups, across, 32, 4, 4), row_fill, dtype=np.uint8)
    r = np.arange(rows)
    full = np.zeros((rows, across * 4), dtype=np.uint8)
    full[:, :blocks] = scales
    for b in range(across * 4):
        out[r // 128, b // 4, r % 32, r // 32 % 4, b % 4] = full[:, b]
    return out.reshape(-1)


def untile_scales(tiled, rows, cols):
    across, groups = ceil_div(cols, 128), ceil_div(rows, 128)
    t = np.asarray(tiled).reshape(groups, across, 32, 4, 4)
    return t.transpose(0, 3, 2, 1, 4).reshape(groups * 128, across * 4)[:rows, :ceil_div(cols, 32)]


def values(codes, scales):
    cols = codes.shape[1]
    scale = np.where(scales == 255, np.nan, np.exp2(scales.astype(np.float64) - 127.0))
    return VALUES[codes] * np.repeat(scale, 32, axis=1)[:, :cols]


def activate(x, act):
    from math import erf, sqrt

    if act == 'none':
        return x
    if act == 'relu':
        return np.where(x < 0, 0.0, x)
    with np.errstate(over='ignore'):
        if act == 'silu':
            return x / (1 + np.exp(-x))
        if act == 'sigmoid':
            return 1 / (1 + np.exp(-x))
    if act == 'gelu':
        return 0.5 * x * (1 + np.vectorize(erf, otypes=[np.float64])(x / sqrt(2)))
    if act == 'gelu_tanh':
        return 0.5 * x * (1 + np.tanh(np.sqrt(2 / np.pi) * (x + 0.044715 * x ** 3)))
    raise ValueError(act)
