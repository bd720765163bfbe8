"""The tail of a decode step, and its scoring: final norm, 8-bit head, and what
follows the logits.

``sample_hidden`` draws one token a row from the residual stream a model's last
layer leaves: :func:`fused_add_rms_norm_fp8` (or :func:`fused_rms_norm_fp8`),
:func:`fp8_linear`, :func:`fused_sample`, three kernels.  ``score_hidden``
scores given tokens with the same head: the norm and the head over chunks of
tokens, so that the logits held stay within 4 GiB, and
:func:`fused_logprob_entropy_forward`; it is what an old-policy or reference
pass needs whose log-probabilities are to match the sampler's.  Neither has a
gradient.
"""
from __future__ import annotations

import torch

from .fp8 import MAX_ROWS, fp8_linear
from .linear_grpo import default_chunk_tokens
from .norm import fused_add_rms_norm_fp8, fused_rms_norm_fp8
from .ops import fused_logprob_entropy_forward
from .sample import fused_sample

__all__ = ["sample_hidden", "score_hidden"]


def _norm(hidden, norm_weight, residual, eps):
    if residual is None:
        return fused_rms_norm_fp8(hidden, norm_weight, eps)
    return fused_add_rms_norm_fp8(hidden, residual, norm_weight, eps)[:2]


def sample_hidden(hidden: torch.Tensor, norm_weight: torch.Tensor, head: torch.Tensor,
                  head_scale: torch.Tensor, uniform: torch.Tensor, temperature=1.0, *,
                  residual: torch.Tensor | None = None, eps: float = 1e-6, top_k=None, top_p=None,
                  min_p=None, logits_dtype: torch.dtype = torch.bfloat16):
    """One token for each row of ``hidden`` ``[..., dim]`` (plus ``residual``,
    of its shape).

    Args:
        norm_weight: ``[dim]`` weight of the final norm, as
            :func:`fused_rms_norm` takes it.
        head, head_scale: ``[V, dim]`` float8_e4m3fn and its scales
            (``quantize_fp8(weight, block_rows=128)``); dim a multiple of 16.
        uniform, temperature, top_k, top_p, min_p: :func:`fused_sample`'s; at
            most 2**20 rows.
        logits_dtype: dtype the logits are rounded to.

    Returns:
        :func:`fused_sample`'s ``(tokens, logp, sample_logp)``, each ``[...]``.
    """
    codes, scales = _norm(hidden, norm_weight, residual, eps)
    logits = fp8_linear(codes, scales, head, head_scale, logits_dtype)
    return fused_sample(logits, uniform, temperature, top_k=top_k, top_p=top_p, min_p=min_p)


def score_hidden(hidden: torch.Tensor, norm_weight: torch.Tensor, head: torch.Tensor,
                 head_scale: torch.Tensor, targets: torch.Tensor,
                 temperature: float | None = None, *, residual: torch.Tensor | None = None,
                 eps: float = 1e-6, logits_dtype: torch.dtype = torch.bfloat16,
                 chunk_tokens: int | None = None):
    """``(logprob, entropy, lse)`` of ``targets`` ``[...]`` under the 8-bit head,
    float32, as :func:`fused_logprob_entropy_forward` gives them for the logits
    that :func:`sample_hidden` draws from (up to the rounding of logits that
    another number of tokens at a time sums in another order).

    Args:
        targets: ``[...]`` int64, ``hidden``'s leading shape.
        chunk_tokens: tokens whose logits are held at a time, at most 2**20 of
            them; by default the fewest equal chunks of at most 4 GiB of logits.
    """
    if targets.dtype != torch.int64:
        raise RuntimeError("targets must be int64")
    if tuple(targets.shape) != tuple(hidden.shape[:-1]):
        raise RuntimeError("hidden[..., D] and targets[...] must have the same leading shape")
    if targets.device != hidden.device:
        raise RuntimeError("hidden and targets must be on the same device")
    if chunk_tokens is not None and chunk_tokens < 1:
        raise ValueError(f"chunk_tokens must be >= 1, got {chunk_tokens}")
    codes, scales = _norm(hidden, norm_weight, residual, eps)
    q, s = codes.reshape(-1, codes.size(-1)), scales.reshape(-1, scales.size(-1))
    t = targets.reshape(-1).contiguous()
    n = t.numel()
    size = 4 if logits_dtype == torch.float32 else 2
    chunk = default_chunk_tokens(n, head.size(0), size) if chunk_tokens is None else chunk_tokens
    chunk = min(chunk, MAX_ROWS)
    out = torch.empty(3, n, dtype=torch.float32, device=hidden.device)
    for i in range(0, n, chunk):
        logits = fp8_linear(q[i:i + chunk], s[i:i + chunk], head, head_scale, logits_dtype)
        for row, part in zip(out, fused_logprob_entropy_forward(logits, t[i:i + chunk],
                                                                temperature)):
            row[i:i + chunk] = part
    return tuple(row.view(targets.shape) for row in out)
