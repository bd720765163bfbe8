"""Float64 statements of the 8-bit operators (numpy): e4m3 quantization with a
scale per block, and the product of two such matrices."""
from __future__ import annotations

import numpy as np

BLOCK = 128
E4M3_MAX = 448.0
MIN_AMAX = 2.0 ** -100


def _e4m3_values():
    """The value of each of the 256 codes (OCP e4m3fn: bias 7, no infinities,
    0x7f and 0xff NaN)."""
    c = np.arange(256)
    sign = np.where(c & 0x80, -1.0, 1.0)
    e, m = (c >> 3) & 15, c & 7
    v = np.where(e == 0, m * 2.0 ** -9, (8 + m) * 2.0 ** (e - 10.0))
    v = np.where((c & 0x7F) == 0x7F, np.nan, v)
    return sign * v


E4M3 = _e4m3_values()


def decode(codes):
    return E4M3[np.asarray(codes, dtype=np.uint8)]


def round_e4m3(x):
    """x (any float array) rounded to the nearest e4m3 value, ties to even;
    magnitudes up to 464 round to 448, beyond that there is none (NaN)."""
    x = np.asarray(x, dtype=np.float64)
    a = np.abs(x)
    with np.errstate(divide="ignore", invalid="ignore"):
        e = np.floor(np.log2(np.maximum(a, 2.0 ** -6)))
        step = 2.0 ** (e - 3)
        r = np.rint(a / step) * step
    r = np.where(a > 464.0, np.nan, np.minimum(r, E4M3_MAX))
    return np.copysign(r, x)


def block_amax(v, block_rows):
    """max |v| per block (NaN where a block holds one)."""
    rows, dim = v.shape
    nr, nd = -(-rows // block_rows), -(-dim // BLOCK)
    p = np.zeros((nr * block_rows, nd * BLOCK), dtype=v.dtype)
    p[:rows, :dim] = np.abs(v)
    return p.reshape(nr, block_rows, nd, BLOCK).max(axis=(1, 3))


def scale_pair(amax):
    """(scale, inverse) of float32 block maxima, in float32 arithmetic."""
    a = np.asarray(amax, dtype=np.float32)
    with np.errstate(divide="ignore", invalid="ignore", over="ignore"):
        c = np.where(a < np.float32(MIN_AMAX), np.float32(MIN_AMAX), a)
        scale = np.where(a == 0, np.float32(1), c / np.float32(E4M3_MAX))
        inv = np.where(a == 0, np.float32(1), np.float32(E4M3_MAX) / c)
    return scale.astype(np.float32), inv.astype(np.float32)


def spread(scales, block_rows, rows, dim):
    """A value per block as one per element."""
    return np.repeat(np.repeat(scales, block_rows, 0)[:rows], BLOCK, 1)[:, :dim]


def quantize(v, block_rows=1):
    """(values, scales) of float32 v: exactly what the operator gives, each
    float32 operation of its formula rounded once."""
    v = np.asarray(v, dtype=np.float32)
    scale, inv = scale_pair(block_amax(v, block_rows))
    with np.errstate(invalid="ignore", over="ignore"):
        z = v * spread(inv, block_rows, *v.shape)
    return round_e4m3(z), scale


def linear(xq, xs, wq, ws):
    """(out, sum of the terms' magnitudes, sum over groups of 8 neighbouring k
    of the largest term's) in float64 of decoded values."""
    x = xq * spread(xs.astype(np.float64), 1, *xq.shape)
    w = wq * spread(ws.astype(np.float64), BLOCK, *wq.shape)
    ax, aw = np.abs(x), np.abs(w)
    largest = np.zeros((x.shape[0], w.shape[0]))
    for k in range(0, x.shape[1], 8):
        top = np.zeros_like(largest)
        for j in range(k, min(k + 8, x.shape[1])):
            np.maximum(top, np.outer(ax[:, j], aw[:, j]), out=top)
        largest += top
    return x @ w.T, ax @ aw.T, largest
