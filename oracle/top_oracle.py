"""Float64 statement of log-probabilities with alternatives and of their
gradient (numpy), one row at a time and in the order of the definition."""
from __future__ import annotations

import math

import numpy as np


def forward_row(x, target, k, temperature=1.0):
    """(logprob, entropy, lse, rank, ids, top_logprob) of a row x; the
    temperature is taken as its float32 value."""
    x = np.asarray(x, dtype=np.float64)
    V = x.size
    t = float(np.float32(temperature))
    ids, top = np.full(k, -1, dtype=np.int64), np.full(k, -math.inf)
    if np.isnan(x).any() or np.isposinf(x).any():
        return math.nan, math.nan, math.nan, -1, ids, np.full(k, math.nan)
    order = np.argsort(-x, kind="stable")
    inside = 0 <= target < V
    rank = int(np.nonzero(order == target)[0][0]) if inside else -1
    if np.isneginf(x).all():
        return math.nan, math.nan, -math.inf, rank, ids, top
    y = (x - x.max()) / t
    w = np.exp(y)
    ln_z = math.log(w.sum())
    p = w / w.sum()
    lse = x.max() / t + ln_z
    entropy = float((p * (ln_z - np.where(p > 0, y, 0.0))).sum())
    logprob = y[target] - ln_z if inside else -lse
    n = min(k, int((~np.isneginf(x)).sum()))
    ids[:n] = order[:n]
    top[:n] = y[order[:n]] - ln_z
    return logprob, entropy, lse, rank, ids, top


def backward_row(x, target, ids, temperature, g_logp=0.0, g_ent=0.0, g_lse=0.0, g_top=None):
    """(d_x, size): the gradient, and per element the magnitudes that its
    rounding errors scale with."""
    x = np.asarray(x, dtype=np.float64)
    t = float(np.float32(temperature))
    y = x / t
    lse = y.max() + math.log(np.exp(y - y.max()).sum())
    lp = np.maximum(y - lse, -1e30)
    p = np.exp(lp)
    entropy = -(p * lp).sum()
    g_top = np.zeros(len(ids)) if g_top is None else np.where(ids >= 0, g_top, 0.0)
    d = p * (g_lse - g_logp - g_top.sum() - g_ent * (lp + entropy))
    size = p * (abs(g_lse) + abs(g_logp) + np.abs(g_top).sum() + abs(g_ent) * (np.abs(lp) + entropy))
    if 0 <= target < x.size:
        d[target] += g_logp
        size[target] += abs(g_logp)
    for i, g in zip(ids, g_top):
        if i >= 0:
            d[i] += g
            size[i] += abs(g)
    return d / t, size / t
