"""Float64 statement of the root-mean-square norm and its gradients (numpy)."""
from __future__ import annotations

import numpy as np


def forward(h, weight, eps):
    """(y, rstd) of the stored rows h."""
    h, weight = np.asarray(h, dtype=np.float64), np.asarray(weight, dtype=np.float64)
    s = 1.0 / np.sqrt((h * h).mean(1, keepdims=True) + eps)
    return h * s * weight, s


def backward(h, weight, eps, g_y, g_h=None):
    """(d_x, d_weight) and the magnitudes their rounding errors scale with:
    per element of d_x |g_h| + s |g_y w| + s^3 |h| sum|g_y w h| / dim, per
    element of d_weight sum |g_y h s|."""
    h, weight = np.asarray(h, dtype=np.float64), np.asarray(weight, dtype=np.float64)
    _, s = forward(h, weight, eps)
    gw = np.asarray(g_y, dtype=np.float64) * weight
    dot = (gw * h).mean(1, keepdims=True)
    d_x = s * (gw - h * s * s * dot)
    size = s * (np.abs(gw) + np.abs(h) * s * s * np.abs(gw * h).mean(1, keepdims=True))
    if g_h is not None:
        d_x = d_x + g_h
        size = size + np.abs(g_h)
    terms = np.asarray(g_y, dtype=np.float64) * h * s
    return d_x, terms.sum(0), size, np.abs(terms).sum(0)
