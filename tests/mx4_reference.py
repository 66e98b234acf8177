"""MXFP4 in numpy, 64 bits: quantisation and the values of codes, written from
the definition (the element nearest to x / scale, ties to the even one)."""
import numpy as np

ELEMENTS = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6])


def quantize(x):
    """codes uint8 [rows][16 blocks] and scales uint8 [rows][blocks] of x
    [rows][dim]."""
    x = np.asarray(x, np.float64)
    rows, dim = x.shape
    blocks = (dim + 31) // 32
    pad = np.zeros((rows, 32 * blocks))
    pad[:, :dim] = x
    b = pad.reshape(rows, blocks, 32)
    codes = np.zeros(b.shape, np.uint8)
    scales = np.zeros((rows, blocks), np.uint8)
    finite = np.isfinite(b).all(2)
    scales[~finite] = 255
    top = np.abs(np.where(finite[:, :, None], b, 0)).max(2)
    exponent = np.where(top > 0, np.frexp(np.where(top > 0, top, 1))[1] - 1, -1000)   # floor(log2)
    unit = np.maximum(exponent - 2, -127)
    scales[finite] = (unit + 127)[finite]
    t = np.where(finite[:, :, None], b, 0) / np.exp2(unit)[:, :, None]
    off = np.abs(np.abs(t)[..., None] - ELEMENTS)
    best = off.min(-1, keepdims=True)
    # of two elements as near, the even one
    rank = np.where(off == best, np.arange(8) % 2, 9)
    codes[:] = rank.argmin(-1).astype(np.uint8) | (np.signbit(t) << 3).astype(np.uint8)
    codes[~finite] = 0
    codes = codes.reshape(rows, -1)
    codes[:, dim:] = 0
    return codes[:, 0::2] | codes[:, 1::2] << 4, scales


def values(codes, scales, dim):
    """float64 [rows][dim] of codes and scales."""
    codes = np.asarray(codes)
    rows, blocks = codes.shape[0], (dim + 31) // 32
    c = np.stack([codes & 15, codes >> 4], 2).reshape(rows, -1)[:, :32 * blocks]
    v = np.where(c & 8, -ELEMENTS[c & 7], ELEMENTS[c & 7])
    s = np.exp2(scales[:, :blocks].astype(np.float64) - 127)
    s[scales[:, :blocks] == 255] = np.nan
    return (v.reshape(rows, blocks, 32) * s[:, :, None]).reshape(rows, -1)[:, :dim]
