"""Sampling: the tokens whose log-probabilities the rest of the package scores.

``fused_sample(logits, uniform, temperature, top_k=, top_p=, min_p=)`` draws
one token a row by inverse transform of a given uniform number and returns the
token with its log-probability under the whole and under the filtered
distribution (csrc/klp_sample.hip: no sort, float64 sums, results that do not
depend on timing; with a top_k, or a min_p and no top_p, the sum behind ``logp``
is of float32 weights).

Per row, with y = (x - max x) / T, w = exp(y) and the vocabulary ordered by
falling x (equal logits by index):
    K: the first ``top_k``;
    P: those of K before which less than ``top_p`` of K's mass lies (the first
       always);
    M: those of P with ``w >= min_p`` (the first always);
    token: the lowest index whose running sum of M's weights, in index order,
       exceeds ``uniform`` times M's mass;
    logp = y - ln(sum of all w): ``fused_logprob_entropy``'s of this token at
       this temperature, up to rounding;
    sample_logp = y - ln(sum of M's w): under the distribution drawn from.
"""
from __future__ import annotations

import math

import torch

from . import _C
from ._library import (DTYPE_CODES, binding, check_status, device_guard, lib, ptr,
                       stream_handle)

__all__ = ["fused_sample"]


def _parameter(value, name, shape, device, dtype, off, low, high):
    """(value, per-row tensor or None) of a parameter given as a number, a
    tensor or None."""
    if value is None:
        return off, None
    if isinstance(value, torch.Tensor):
        if value.device != device or tuple(value.shape) != tuple(shape):
            raise RuntimeError(f"{name} must be a number or {tuple(shape)} on {device}, got "
                               f"{tuple(value.shape)} on {value.device}")
        if dtype == torch.int32 and value.is_floating_point():
            raise RuntimeError(f"{name} must hold integers")
        if dtype == torch.int32 and value.dtype == torch.int64:
            value = value.clamp(0, 2 ** 31 - 1)
        return off, value.detach().to(dtype).contiguous()
    if dtype == torch.int32:
        # value - value: NaN for an infinity or a NaN.
        if isinstance(value, bool) or value - value != 0 or int(value) != value:
            raise ValueError(f"{name} must be an integer, got {value!r}")
        value = int(value)
    else:
        value = float(value)
    if not low <= value <= high or math.isinf(value):
        raise ValueError(f"{name} must be in [{low}, {high}], got {value}")
    return value, None


def fused_sample(logits: torch.Tensor, uniform: torch.Tensor, temperature=1.0, *, top_k=None,
                 top_p=None, min_p=None):
    """Draw one token a row.

    Args:
        logits: ``[..., V]`` bf16 / fp16 / fp32 on the GPU, any layout
            :func:`kernel_opt.fused_logprob_entropy` takes; -inf logits have
            no weight.  V at most 2**26.
        uniform: ``[...]`` float32 in [0, 1), such as ``torch.rand``'s.
        temperature: T >= 0; 0 takes the largest logit (the lowest index of
            equal ones), with ``logp`` at T = 1 and ``sample_logp`` 0.
        top_k, top_p, min_p: filters, in this order; None turns one off, and
            so do ``top_k`` <= 0 or >= V, ``top_p`` 1 and ``min_p`` 0.

    Every parameter is a number or a tensor shaped like ``uniform`` with one
    value a row (read as float32, ``top_k`` as int32).  A number that is not in
    range raises ValueError: T >= 0 and finite, ``top_k`` an integer, ``top_p``
    and ``min_p`` in [0, 1].  A tensor's values are not checked: a row whose
    temperature is negative or not finite gets token -1, as do rows without a
    distribution, below; a ``top_p`` above 1 and a ``min_p`` below 0, or a NaN
    of either, is off, a ``top_p`` below 0 counts as 0, a ``min_p`` above 1 as 1.

    Returns:
        ``(tokens, logp, sample_logp)``, int64 and twice float32, each
        ``[...]``.  A row of -inf logits gives (-1, -inf, -inf); one with a NaN
        or +inf logit (-1, NaN, NaN).  There is no gradient.
    """
    if not (logits.is_cuda and uniform.is_cuda):
        raise RuntimeError("logits and uniform must be GPU tensors")
    rows = _C.row_layout(logits)
    if rows is None:
        raise RuntimeError("logits must be contiguous")
    if logits.dtype not in DTYPE_CODES:
        raise RuntimeError("logits dtype must be bf16, fp16, or fp32")
    if logits.size(-1) < 1:
        raise RuntimeError("logits last dim (vocab) must be >= 1")
    shape, dev = uniform.shape, logits.device
    if uniform.dtype != torch.float32 or uniform.device != dev \
            or tuple(shape) != tuple(logits.shape[:-1]):
        raise RuntimeError(f"uniform must be float32 {tuple(logits.shape[:-1])} on {dev}, got "
                           f"{uniform.dtype} {tuple(shape)} on {uniform.device}")
    inf = math.inf
    t, ts = _parameter(temperature, "temperature", shape, dev, torch.float32, 1.0, 0.0, inf)
    k, ks = _parameter(top_k, "top_k", shape, dev, torch.int32, 0, -inf, inf)
    k = min(max(k, 0), 2 ** 31 - 1)
    p, ps = _parameter(top_p, "top_p", shape, dev, torch.float32, 1.0, 0.0, 1.0)
    m, ms = _parameter(min_p, "min_p", shape, dev, torch.float32, 0.0, 0.0, 1.0)
    try:
        return tuple(binding.sample(logits, uniform, t, ts, k, ks, p, ps, m, ms))
    except binding.CaptureDeclined:
        pass
    u = uniform.detach().contiguous()
    tokens = torch.empty(shape, dtype=torch.int64, device=dev)
    logp = torch.empty(shape, dtype=torch.float32, device=dev)
    sample_logp = torch.empty(shape, dtype=torch.float32, device=dev)
    with device_guard(dev.index):
        check_status(lib.klp_sample(
            ptr(logits), DTYPE_CODES[logits.dtype], u.numel(), logits.size(-1), *rows, ptr(u), t,
            ptr(ts), k, ptr(ks), p, ptr(ps), m, ptr(ms), ptr(tokens), ptr(logp), ptr(sample_logp),
            stream_handle(dev.index)))
    return tokens, logp, sample_logp
