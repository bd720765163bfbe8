"""Float64 statement of the norms around a block, its gate and residual scale,
and of their gradients (numpy).  Gates come broadcast to the rows (1 without)."""
from __future__ import annotations

import numpy as np


def rstd(v, eps):
    v = np.asarray(v, dtype=np.float64)
    return 1.0 / np.sqrt((v * v).mean(1, keepdims=True) + eps)


def forward(x, residual, post, gate, scale, eps):
    """(h before its rounding, the branch's part of it)."""
    x = np.asarray(x, dtype=np.float64)
    z = x if post is None else x * rstd(x, eps) * post
    u = scale * gate * z
    return residual + u, u


def backward(x, h, s_x, s_h, weight, post, gate, scale, g_y, g_h, unit):
    """Gradients of rows x, h with statistics s_x, s_h (those of the stored
    rows), and bounds of their float32 errors before the final rounding.

    ``unit`` is (srel, sums, half): the relative error of a statistic, that of a
    row's sum and the products around it, and half a step of float32.
    Returns {name: (value, error)} per element (d_gate: per row and element)."""
    srel, sums, half = unit
    rows = x.shape[0]
    gw = g_y * weight
    mean = lambda v: v.mean(1, keepdims=True)  # noqa: E731
    d_h = g_h + s_h * (gw - h * s_h ** 2 * mean(gw * h))
    size = np.abs(g_h) + s_h * (np.abs(gw) + np.abs(h) * s_h ** 2 * mean(np.abs(gw * h)))
    e_h = size * (3 * srel + sums)
    d_z = scale * gate * d_h
    e_z = np.abs(scale * gate) * e_h + 3 * half * np.abs(d_z)
    out = {"residual": (d_h, e_h)}
    if post is None:
        z = x
        out["x"] = (d_z, e_z)
    else:
        z = x * s_x * post
        gp = d_z * post
        e_p = np.abs(post) * e_z + half * np.abs(gp)
        d_x = s_x * (gp - x * s_x ** 2 * mean(gp * x))
        size = s_x * (np.abs(gp) + np.abs(x) * s_x ** 2 * mean(np.abs(gp * x)))
        e_x = s_x * (e_p + np.abs(x) * s_x ** 2 * mean(e_p * np.abs(x))) + size * (3 * srel + sums)
        out["x"] = (d_x, e_x)
    many = srel + (rows + 24) * half
    terms = g_y * h * s_h
    out["weight"] = (terms.sum(0), np.abs(terms).sum(0) * many)
    if post is not None:
        terms = d_z * x * s_x
        out["post"] = (terms.sum(0), (np.abs(terms) * many + e_z * np.abs(x) * s_x).sum(0))
    terms = scale * z * d_h
    out["gate"] = (terms, np.abs(terms) * (2 * srel + many) + np.abs(scale * z) * e_h)
    return out
