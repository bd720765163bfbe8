"""The norms around a block: its output through a norm, a gate and a residual
scale into the residual stream, and the next block's norm.

``fused_block_norm(x, residual, weight, post_weight=, gate=, scale=)`` computes,
per row of ``dim`` elements,

    z = x * (mean(x^2) + eps)^-1/2 * post_weight     (z = x without one)
    h = round(residual + scale * gate * z)           (gate 1 without one)
    y = round(h * (mean(h^2) + eps)^-1/2 * weight)

in one pass (csrc/klp_block.hip), differentiable in every tensor.  Without
``post_weight``, ``gate`` and ``scale`` it is :func:`fused_add_rms_norm`.  All
sums are float32; ``h`` and ``y`` are rounded once.  The gradient is of first
order: a second derivative raises RuntimeError.

With ``checkpoint="fp8"`` the forward keeps ``x`` and ``h`` for the backward as
e4m3 codes with a float32 scale for each 128 columns (:func:`quantize_fp8`'s),
2.06 bytes an element instead of 4, and the gradients' formulas take the values
that the codes stand for; the outputs and the statistics are the exact ones
(``create_graph`` raises RuntimeError).

``fused_block_norm_fp8`` writes ``y`` as e4m3 codes and scales, the operand of
:func:`fp8_linear` (serving: no gradient).

Calls run in the compiled binding (binding/klp_torch.cpp), the autograd function
included; under graph capture, which it declines, the Python statement of them
below runs.  ``torch.compile`` breaks the graph at a call and runs it as it is
(:func:`fused_add_rms_norm` is traced).
"""
from __future__ import annotations

import math

import torch

from ._library import (DTYPE_CODES, binding, check_status, device_guard, lib, ptr,
                       stream_handle)
from ._order import first_order
from .norm import SCALE_BLOCK, _rows

__all__ = ["fused_block_norm", "fused_block_norm_fp8"]

MAX_DIM = 16384


def _rows_per_gate(x, gate):
    """Consecutive rows of ``x`` that share a row of ``gate``; None where it
    does not fit."""
    n = x.numel() // x.size(-1)
    if gate.dim() == 1:
        return max(n, 1)
    if gate.dim() != x.dim():
        return None
    lead, of = gate.shape[:-1], x.shape[:-1]
    same = 0
    while same < len(of) and lead[same] == of[same]:
        same += 1
    if any(s != 1 for s in lead[same:]):
        return None
    return max(math.prod(of[same:]), 1)


def _check(x, residual, weight, post_weight, gate, scale, eps):
    """(rows that share a gate, scale as a number)."""
    if not x.is_cuda:
        raise RuntimeError("x must be a GPU tensor")
    if x.dtype not in DTYPE_CODES:
        raise RuntimeError("x must be bf16, fp16, or fp32")
    if x.dim() < 1 or not 1 <= x.size(-1) <= MAX_DIM:
        raise RuntimeError(f"the last dim of x must be in [1, {MAX_DIM}], got {tuple(x.shape)}")
    D = x.size(-1)
    if residual.device != x.device or residual.dtype != x.dtype or residual.shape != x.shape:
        raise RuntimeError("residual must have x's shape, dtype and device")
    for name, w in (("weight", weight), ("post_weight", post_weight)):
        if w is None and name == "post_weight":
            continue
        if w.device != x.device or tuple(w.shape) != (D,):
            raise RuntimeError(f"{name} must be [{D}] on {x.device}, got {tuple(w.shape)} on "
                               f"{w.device}")
        if w.dtype not in (x.dtype, torch.float32) or w.dtype != weight.dtype:
            raise RuntimeError("weight and post_weight must both be float32 or of x's dtype")
    per_gate = 1
    if gate is not None:
        if gate.device != x.device or gate.dtype not in (x.dtype, torch.float32):
            raise RuntimeError(f"gate must be float32 or of x's dtype, on {x.device}")
        per_gate = _rows_per_gate(x, gate) if gate.dim() and gate.size(-1) == D else None
        if per_gate is None:
            raise RuntimeError(f"gate must be [{D}] or x's shape {tuple(x.shape)} with 1 in place "
                               f"of the last leading dims, got {tuple(gate.shape)}")
    scale = float(scale)
    if not math.isfinite(scale):
        raise RuntimeError(f"scale must be finite, got {scale}")
    if not (eps >= 0.0 and eps != float("inf")):
        raise RuntimeError(f"eps must be finite and >= 0, got {eps}")
    return per_gate, scale


def _code(t):
    return 0 if t is None else DTYPE_CODES[t.dtype]


def _codes_like(x):
    return (torch.empty(x.shape, dtype=torch.float8_e4m3fn, device=x.device),
            torch.empty(*x.shape[:-1], -(-x.size(-1) // SCALE_BLOCK), dtype=torch.float32,
                        device=x.device))


def _operands(x, residual, weight, post, gate):
    x2, ld_x = _rows(x)
    r2, ld_r = _rows(residual)
    return x2, ld_x, r2, ld_r, weight.contiguous(), \
        None if post is None else post.contiguous(), None if gate is None else gate.contiguous()


class _FusedBlockNorm(torch.autograd.Function):

    @staticmethod
    def forward(ctx, x, residual, weight, post, gate, per_gate, scale, eps, kept):
        dev = x.device
        x2, ld_x, r2, ld_r, w, wp, g = _operands(x, residual, weight, post, gate)
        N, D = x2.shape
        y, h = (torch.empty(x.shape, dtype=x.dtype, device=dev) for _ in range(2))
        rstd_x, rstd_h = (torch.empty(N, dtype=torch.float32, device=dev) for _ in range(2))
        needs_x = post is not None or gate is not None
        xq, xs = _codes_like(x) if kept and needs_x else (None, None)
        hq, hs = _codes_like(x) if kept else (None, None)
        with device_guard(dev.index):
            check_status(lib.klp_block_norm(
                ptr(x2), _code(x), ld_x, ptr(r2), ld_r, ptr(wp), ptr(w), _code(w), ptr(g),
                _code(g), per_gate, scale, N, D, eps, ptr(y), ptr(h), ptr(rstd_x), ptr(rstd_h),
                ptr(xq), ptr(xs), ptr(hq), ptr(hs), stream_handle(dev.index)))
        ctx.save_for_backward(x if needs_x and not kept else None, None if kept else h, xq, xs, hq,
                              hs, weight, post, gate, rstd_x, rstd_h)
        ctx.how = per_gate, scale
        ctx.like = x.shape, x.dtype, dev
        ctx.set_materialize_grads(False)
        return y, h

    @staticmethod
    def backward(ctx, g_y, g_h):
        x, h, xq, xs, hq, hs, weight, post, gate, rstd_x, rstd_h = ctx.saved_tensors
        per_gate, scale = ctx.how
        shape, dtype, dev = ctx.like
        need = ctx.needs_input_grad[:5]
        if (g_y is None and g_h is None) or not any(need):
            return (None,) * 9
        if hq is not None and torch.is_grad_enabled():
            raise RuntimeError("kernel_opt: gradients from 8-bit checkpoints cannot be "
                               "differentiated (create_graph)")

        def new(t, wanted):
            return None if t is None or not wanted else torch.empty(t.shape, dtype=t.dtype,
                                                                    device=dev)

        D = shape[-1]
        N = math.prod(shape[:-1])
        plain = post is None and gate is None and scale == 1.0  # then d_x is d_residual
        d_x, d_r = (torch.empty(shape, dtype=dtype, device=dev) if n else None
                    for n in (need[0] and not (plain and need[1]), need[1]))
        d_w, d_p, d_g = (new(t, n) for t, n in zip((weight, post, gate), need[2:]))
        if N == 0:
            for t in (d_w, d_p, d_g):
                if t is not None:
                    t.zero_()
        else:
            gy, gh = (None if g is None else g.contiguous() for g in (g_y, g_h))
            x2, ld_x = (None, 0) if x is None else _rows(x)
            w, wp, g = (None if t is None else t.contiguous() for t in (weight, post, gate))
            nbytes = 0
            if d_w is not None or d_p is not None or d_g is not None:
                nbytes = lib.klp_block_norm_bwd_workspace_bytes(N, D, post is not None,
                                                                gate is not None, per_gate)
            ws = torch.empty(nbytes, dtype=torch.uint8, device=dev) if nbytes else None
            with device_guard(dev.index):
                check_status(lib.klp_block_norm_bwd(
                    ptr(x2), DTYPE_CODES[dtype], ld_x, ptr(xq), ptr(xs), ptr(h), ptr(hq), ptr(hs),
                    ptr(wp), ptr(w), _code(w), ptr(g), _code(g), per_gate, scale, ptr(rstd_x),
                    ptr(rstd_h), ptr(gy), ptr(gh), N, D, ptr(d_x), ptr(d_r), ptr(d_p), ptr(d_w),
                    ptr(d_g), ptr(ws), nbytes, stream_handle(dev.index)))
        if plain and need[0] and need[1]:
            d_x = d_r
        grads = first_order("fused_block_norm", (d_x, d_r, d_w, d_p, d_g),
                            (x, h, weight, post, gate, g_y, g_h))
        return (*grads, None, None, None, None)


def fused_block_norm(x: torch.Tensor, residual: torch.Tensor, weight: torch.Tensor, *,
                     post_weight: torch.Tensor | None = None, gate: torch.Tensor | None = None,
                     scale: float = 1.0, eps: float = 1e-6, checkpoint: str | None = None):
    """``(y, h)``: the residual stream ``h`` behind a block whose output is
    ``x``, and its norm ``y`` for the next one.

    Args:
        x, residual: ``[..., dim]`` bf16 / fp16 / fp32 on the GPU, dim at most
            16384, fewer than 2**22 rows (RuntimeError otherwise).
        weight, post_weight: ``[dim]``, both of ``x``'s dtype or both float32.
        gate: ``[dim]``, or ``x``'s shape with 1 in place of the last leading
            dims (``[batch, 1, dim]`` gates each sequence), of ``x``'s dtype or
            float32.
        scale: the residual scale, a finite number.
        checkpoint: "fp8" keeps ``x`` and ``h`` for the backward in 8 bits.
    """
    per_gate, scale = _check(x, residual, weight, post_weight, gate, scale, eps)
    if checkpoint not in (None, "fp8"):
        raise ValueError(f'checkpoint must be None or "fp8", got {checkpoint!r}')
    kept = checkpoint is not None and torch.is_grad_enabled() and any(
        t is not None and t.requires_grad for t in (x, residual, weight, post_weight, gate))
    args = (x, residual, weight, post_weight, gate, per_gate, scale, float(eps), kept)
    try:
        return tuple(binding.block_norm(*args))
    except binding.CaptureDeclined:
        return _FusedBlockNorm.apply(*args)


def fused_block_norm_fp8(x: torch.Tensor, residual: torch.Tensor, weight: torch.Tensor, *,
                         post_weight: torch.Tensor | None = None,
                         gate: torch.Tensor | None = None, scale: float = 1.0,
                         eps: float = 1e-6):
    """``(codes, scales, h)``: :func:`fused_block_norm`'s unrounded ``y`` as
    :func:`fused_rms_norm_fp8` writes it, and ``h``.  No gradient: the outputs
    are detached from inputs that require one."""
    per_gate, scale = _check(x, residual, weight, post_weight, gate, scale, eps)
    try:
        return tuple(binding.block_norm_fp8(x, residual, weight, post_weight, gate, per_gate, scale,
                                            float(eps)))
    except binding.CaptureDeclined:
        pass
    x, residual, weight, post_weight, gate = (
        None if t is None else t.detach() for t in (x, residual, weight, post_weight, gate))
    dev = x.device
    x2, ld_x, r2, ld_r, w, wp, g = _operands(x, residual, weight, post_weight, gate)
    h = torch.empty(x.shape, dtype=x.dtype, device=dev)
    q, scales = _codes_like(x)
    with device_guard(dev.index):
        check_status(lib.klp_block_norm_fp8(
            ptr(x2), _code(x), ld_x, ptr(r2), ld_r, ptr(wp), ptr(w), _code(w), ptr(g), _code(g),
            per_gate, scale, x2.size(0), x2.size(1), float(eps), ptr(q), ptr(scales), ptr(h),
            stream_handle(dev.index)))
    return q, scales, h
