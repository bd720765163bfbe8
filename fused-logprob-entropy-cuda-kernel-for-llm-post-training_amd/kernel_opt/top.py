"""Log-probabilities of given tokens with their alternatives.

``fused_top_logprobs(logits, targets, k)`` reads each row of logits once and
returns, beside ``fused_logprob_entropy``'s three numbers, the target's rank
and the k most likely tokens with their log-probabilities (csrc/klp_top.hip).
Per row, with y = x / T and the vocabulary ordered by falling x (equal logits
by index):

    logprob = y[target] - lse,  entropy = lse - sum p y,  lse = ln sum exp(y)
    rank = tokens before the target in the order (0: the most likely one)
    top_ids = the order's first k,  top_logprob = y[top_ids] - lse

Differentiable in ``logits`` through the four kinds of log-probability, with
one pass that reads the logits and writes their gradient: what a distillation
loss over a student's likely tokens needs beside its policy terms.  The
gradient is of first order: a second derivative raises RuntimeError.

Calls run in the compiled binding (binding/klp_torch.cpp), the autograd
function included; under graph capture, which it declines, the Python statement
of them below runs.  ``torch.compile`` breaks the graph at a call and runs it as it
is.
"""
from __future__ import annotations

import math

import torch

from . import _C
from ._library import (DTYPE_CODES, binding, capturing, check_status, device_guard,
                       keep_for_capture, lib, ptr, stream_handle)
from ._order import first_order

__all__ = ["fused_top_logprobs"]

MAX_K = 256
MAX_VOCAB = 2 ** 26


def _check(logits, targets, k, temperature):
    """(k, T) as numbers."""
    if not (logits.is_cuda and targets.is_cuda):
        raise RuntimeError("logits and targets must be GPU tensors")
    if logits.dtype not in DTYPE_CODES:
        raise RuntimeError("logits dtype must be bf16, fp16, or fp32")
    if logits.dim() < 1 or not 1 <= logits.size(-1) <= MAX_VOCAB:
        raise RuntimeError(f"logits last dim (vocab) must be in [1, 2**26], got "
                           f"{tuple(logits.shape)}")
    if _C.row_layout(logits) is None:
        raise RuntimeError("logits must be contiguous")
    if targets.dtype != torch.int64:
        raise RuntimeError("targets must be int64")
    if targets.device != logits.device or targets.shape != logits.shape[:-1]:
        raise RuntimeError(f"targets must be {tuple(logits.shape[:-1])} on {logits.device}, got "
                           f"{tuple(targets.shape)} on {targets.device}")
    if isinstance(k, bool) or int(k) != k or not 1 <= k <= MAX_K:
        raise ValueError(f"k must be an integer in [1, {MAX_K}], got {k!r}")
    t = 1.0 if temperature is None else float(temperature)
    if not t > 0.0 or math.isinf(t):
        raise RuntimeError(f"temperature must be finite and > 0, got {t}")
    return int(k), t


def _forward(logits, targets, k, temperature):
    """The six outputs in new dense tensors, under graph capture."""
    dev = logits.device
    t = targets.contiguous()
    f32 = dict(dtype=torch.float32, device=dev)
    logprob, entropy, lse = (torch.empty(t.shape, **f32) for _ in range(3))
    rank = torch.empty(t.shape, dtype=torch.int64, device=dev)
    ids = torch.empty(*t.shape, k, dtype=torch.int64, device=dev)
    top = torch.empty(*t.shape, k, **f32)
    N, V = t.numel(), logits.size(-1)
    code = DTYPE_CODES[logits.dtype]
    nbytes = lib.klp_fwd_top_workspace_bytes(code, N, V, k)
    ws = None
    if nbytes:  # a call's own: zero before its first use, kept as long as its graph may be
        ws = torch.empty(nbytes, dtype=torch.uint8, device=dev).zero_()
        if capturing():
            keep_for_capture(ws)
    with device_guard(dev.index):
        check_status(lib.klp_fwd_top(
            ptr(logits), code, N, V, *_C.row_layout(logits), ptr(t), temperature, k, ptr(logprob),
            ptr(entropy), ptr(lse), ptr(rank), ptr(ids), ptr(top), ptr(ws), nbytes,
            stream_handle(dev.index)))
    return logprob, entropy, lse, rank, ids, top


class _FusedTopLogprobs(torch.autograd.Function):

    @staticmethod
    def forward(ctx, logits, targets, k, temperature):
        out = _forward(logits, targets, k, temperature)
        ctx.save_for_backward(logits, targets, out[1], out[2], out[4])
        ctx.temperature = temperature
        ctx.mark_non_differentiable(out[3], out[4])
        ctx.set_materialize_grads(False)
        return out

    @staticmethod
    def backward(ctx, g_logp, g_ent, g_lse, _g_rank, _g_ids, g_top):
        logits, targets, entropy, lse, ids = ctx.saved_tensors
        given = (g_logp, g_ent, g_lse, g_top)
        if not ctx.needs_input_grad[0] or all(g is None for g in given):
            return None, None, None, None
        dev = logits.device
        gl, ge, gs, gt = (None if g is None else g.to(torch.float32).contiguous() for g in given)
        t = targets.contiguous()
        d = torch.empty(logits.shape, dtype=logits.dtype, device=dev)
        with device_guard(dev.index):
            check_status(lib.klp_bwd_top(
                ptr(logits), DTYPE_CODES[logits.dtype], t.numel(), logits.size(-1),
                *_C.row_layout(logits), ptr(t), ctx.temperature, ids.size(-1), ptr(ids), ptr(lse),
                ptr(entropy), ptr(gl), ptr(ge), ptr(gs), ptr(gt), ptr(d),
                stream_handle(dev.index)))
        d, = first_order("fused_top_logprobs", (d,), (logits, *given))
        return d, None, None, None


def fused_top_logprobs(logits: torch.Tensor, targets: torch.Tensor, k: int,
                       temperature: float | None = None):
    """Log-probabilities of ``targets`` and of the ``k`` most likely tokens.

    Args:
        logits: ``[..., V]`` bf16 / fp16 / fp32 on the GPU, any layout
            :func:`kernel_opt.fused_logprob_entropy` takes; V at most 2**26, fewer
            than 2**23 rows (RuntimeError otherwise).
        targets: ``[...]`` int64.  One outside [0, V), an ignore index, has
            logprob -lse (as :func:`fused_logprob_entropy` gives it) and rank -1.
        k: alternatives of a row, 1 to 256.
        temperature: T > 0; None is 1.

    Returns:
        ``(logprob, entropy, lse, rank, top_ids, top_logprob)``: ``[...]``
        float32 three times and int64, ``[..., k]`` int64 and float32, likeliest
        first, equal logits by index.  Logits of -inf are not listed: places left
        over hold -1 and -inf.  A row with a NaN or +inf logit has rank and
        top_ids -1 and NaN otherwise; one of -inf logits only has lse -inf, and
        logprob and entropy NaN.  Finite logits are right at any size, as far as
        float32 holds the result: a row masked as a whole with a finite fill is
        uniform.
    """
    k, t = _check(logits, targets, k, temperature)
    try:
        return tuple(binding.top_logprobs(logits, targets, k, t))
    except binding.CaptureDeclined:
        return _FusedTopLogprobs.apply(logits, targets, k, t)
