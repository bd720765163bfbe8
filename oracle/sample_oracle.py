"""Float64 statement of sampling with temperature, top-k, top-p and min-p
(numpy), one row at a time and in the order of the definition."""
from __future__ import annotations

import math

import numpy as np


def sample_row(x, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """(token, logp, sample_logp, kept indices) of one row.  Parameters are
    taken as their float32 values."""
    x = np.asarray(x, dtype=np.float64)
    V = x.size
    t, top_p, min_p = (float(np.float32(v)) for v in (temperature, top_p, min_p))
    none = np.zeros(0, dtype=np.int64)
    if np.isnan(x).any() or np.isposinf(x).any() or not (t >= 0 and math.isfinite(t)):
        return -1, math.nan, math.nan, none
    if np.isneginf(x).all():
        return -1, -math.inf, -math.inf, none
    if t == 0.0:
        t, top_k = 1.0, 1
    y = (x - x.max()) / t
    w = np.exp(y)
    order = np.argsort(-x, kind="stable")
    if 0 < top_k < V:
        order = order[:top_k]
    if top_p < 1.0:
        ws = w[order]
        before = np.concatenate([[0.0], np.cumsum(ws)[:-1]])
        keep = before < max(top_p, 0.0) * ws.sum()
        keep[0] = True
        order = order[keep]
    if min_p > 0.0:
        keep = w[order] >= min(min_p, 1.0)
        keep[0] = True
        order = order[keep]
    kept = np.sort(order)
    run = np.cumsum(w[kept])
    u = min(max(float(np.float32(u)), 0.0), 1.0) if u == u else 0.0
    past = np.nonzero(run > u * run[-1])[0]
    at = past[0] if past.size else np.nonzero(w[kept] > 0)[0][-1]
    token = int(kept[at])
    return token, y[token] - math.log(w.sum()), y[token] - math.log(run[-1]), kept
