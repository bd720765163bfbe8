"""Root-mean-square norm in front of the LM head, with the residual's addition.

``fused_rms_norm(x, weight)`` and ``fused_add_rms_norm(x, residual, weight)``
compute, per row of ``dim`` elements,

    h = round(x + residual)                   (h = x without a residual)
    y = round(h * (mean(h^2) + eps)^-1/2 * weight)

in one pass (csrc/klp_norm.hip), differentiable in ``x``, ``residual`` and
``weight``: the backward reads ``h`` and one float32 a row.  The gradient is of
first order: with ``create_graph=True`` a second derivative through it raises
RuntimeError (what flows through ``h`` alone has one).  The statistics are
those of the stored ``h``, all sums are float32, ``y`` is rounded once; a row
whose sum of squares passes float32's range gives zeros.

``fused_rms_norm_fp8`` / ``fused_add_rms_norm_fp8`` write the same ``y`` as
e4m3 codes with a float32 scale for each 128 columns, the operand of
:func:`kernel_opt.fp8_linear` (serving and scoring: no gradient).

Calls run in the compiled binding (binding/klp_torch.cpp), the autograd function
included; under graph capture, which it declines, the Python statement of them
below runs, and under ``torch.compile`` the two differentiable ones go through
the registered op ``torch.ops.kernel_opt.rms_norm`` (no graph break).
"""
from __future__ import annotations

import torch

from ._library import (DTYPE_CODES, binding, check_status, device_guard, lib, ptr,
                       stream_handle)

__all__ = ["fused_rms_norm", "fused_add_rms_norm", "fused_rms_norm_fp8", "fused_add_rms_norm_fp8"]

SCALE_BLOCK = 128
MAX_DIM = 65536


def _check(x, residual, weight, eps):
    if not x.is_cuda:
        raise RuntimeError("x must be a GPU tensor")
    if x.dtype not in DTYPE_CODES:
        raise RuntimeError("x must be bf16, fp16, or fp32")
    if x.dim() < 1:
        raise RuntimeError("x must have at least one dimension")
    D = x.size(-1)
    if not 1 <= D <= MAX_DIM:
        raise RuntimeError(f"the last dim of x must be in [1, {MAX_DIM}], got {D}")
    if weight.device != x.device or tuple(weight.shape) != (D,):
        raise RuntimeError(f"weight must be [{D}] on {x.device}, got {tuple(weight.shape)} on "
                           f"{weight.device}")
    if weight.dtype not in (x.dtype, torch.float32):
        raise RuntimeError("weight must be float32 or of x's dtype")
    if residual is not None:
        if residual.device != x.device or residual.dtype != x.dtype or residual.shape != x.shape:
            raise RuntimeError("residual must have x's shape, dtype and device")
    if not (eps >= 0.0 and eps != float("inf")):
        raise RuntimeError(f"eps must be finite and >= 0, got {eps}")


def _rows(t):
    """``t`` as rows of its last dim with unit stride (a view where its layout
    has one) and their stride."""
    t2 = t.reshape(-1, t.size(-1))
    if t2.size(-1) > 1 and t2.stride(-1) != 1:
        t2 = t2.contiguous()
    return t2, t2.stride(0) if t2.size(0) > 1 else t2.size(1)


def _forward(x, residual, weight, eps, fp8):
    """(y or (codes, scales), h or None, rstd or None) into new dense tensors."""
    dev = x.device
    D = x.size(-1)
    x2, ld_x = _rows(x)
    r2, ld_r = (None, 0) if residual is None else _rows(residual)
    w = weight.contiguous()
    N = x2.size(0)
    h = None if residual is None else torch.empty(x.shape, dtype=x.dtype, device=dev)
    args = [ptr(x2), DTYPE_CODES[x.dtype], ld_x, ptr(r2), ld_r, ptr(w), DTYPE_CODES[w.dtype], N, D,
            float(eps)]
    if fp8:
        q = torch.empty(x.shape, dtype=torch.float8_e4m3fn, device=dev)
        scales = torch.empty(*x.shape[:-1], -(-D // SCALE_BLOCK), dtype=torch.float32, device=dev)
        with device_guard(dev.index):
            check_status(lib.klp_rms_norm_fp8(*args, ptr(q), ptr(scales), ptr(h),
                                              stream_handle(dev.index)))
        return (q, scales), h, None
    y = torch.empty(x.shape, dtype=x.dtype, device=dev)
    rstd = torch.empty(N, dtype=torch.float32, device=dev)
    with device_guard(dev.index):
        check_status(lib.klp_rms_norm(*args, ptr(y), ptr(h), ptr(rstd), stream_handle(dev.index)))
    return y, h, rstd


def _backward(h, weight, rstd, g_y, g_h, need_w):
    """(d_x, d_weight or None) into new dense tensors."""
    dev = h.device
    h2, ld_h = _rows(h)
    N, D = h2.shape
    d_x = torch.empty(h.shape, dtype=h.dtype, device=dev)
    d_w = torch.empty_like(weight, memory_format=torch.contiguous_format) if need_w else None
    if N == 0:
        return d_x, d_w.zero_() if need_w else None
    g_y = g_y.contiguous()
    g_h = None if g_h is None else g_h.contiguous()
    nbytes = lib.klp_rms_norm_bwd_workspace_bytes(N, D) if need_w else 0
    ws = torch.empty(nbytes, dtype=torch.uint8, device=dev) if need_w else None
    w = weight.contiguous()
    with device_guard(dev.index):
        check_status(lib.klp_rms_norm_bwd(
            ptr(h2), DTYPE_CODES[h.dtype], ld_h, ptr(w), DTYPE_CODES[w.dtype], ptr(rstd),
            ptr(g_y), ptr(g_h), N, D, ptr(d_x), ptr(d_w), ptr(ws), nbytes,
            stream_handle(dev.index)))
    return d_x, d_w


class _FirstOrder(torch.autograd.Function):
    """The norm's gradients as functions of what they depend on (``of``), whose
    own gradient is refused: left without a graph they would count as constants
    in a second derivative."""

    @staticmethod
    def forward(ctx, d_x, d_w, *of):
        return d_x, d_w

    @staticmethod
    def backward(ctx, *grads):
        raise RuntimeError("kernel_opt: the root-mean-square norms have no second derivative")


def _gradients(ctx, g_y, g_h, backward):
    """Gradients of (x, residual, weight), by ``backward`` where y's is given."""
    h, weight, rstd = ctx.saved_tensors
    need_x, need_r, need_w = ctx.needs_input_grad[:3]
    if (g_y is None and g_h is None) or not (need_x or need_r or need_w):
        return None, None, None
    if g_y is None:  # only h was used
        d_w = torch.zeros_like(weight) if need_w else None
        return g_h if need_x else None, g_h if need_r else None, d_w
    d_x, d_w = backward(h, weight, rstd, g_y, g_h, need_w)
    return d_x if need_x else None, d_x if need_r else None, d_w


class _FusedRmsNorm(torch.autograd.Function):

    @staticmethod
    def forward(ctx, x, residual, weight, eps):
        y, h, rstd = _forward(x, residual, weight, eps, False)
        ctx.save_for_backward(x if h is None else h, weight, rstd)
        ctx.set_materialize_grads(False)
        return y if h is None else (y, h)

    @staticmethod
    def backward(ctx, g_y, g_h=None):
        def first_order(h, weight, rstd, g_y, g_h, need_w):
            d_x, d_w = _backward(h, weight, rstd, g_y, g_h, need_w)
            if torch.is_grad_enabled():  # create_graph
                d_x, d_w = _FirstOrder.apply(d_x, d_w, h, weight, g_y, g_h)
            return d_x, d_w

        return *_gradients(ctx, g_y, g_h, first_order), None


# ---------------------------------------------------------------------------
# torch.library registration, for torch.compile: the norm traces without a
# graph break.  Eager calls take the compiled autograd function.
# ---------------------------------------------------------------------------
@torch.library.custom_op("kernel_opt::rms_norm", mutates_args=(), device_types="cuda")
def _op_forward(x: torch.Tensor, residual: torch.Tensor | None, weight: torch.Tensor,
                eps: float) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    y, h, rstd = _forward(x, residual, weight, eps, False)
    return y, x.new_empty(0) if h is None else h, rstd


@_op_forward.register_fake
def _(x, residual, weight, eps):
    y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    rstd = x.new_empty(x.numel() // x.size(-1), dtype=torch.float32)
    return y, x.new_empty(0) if residual is None else torch.empty_like(y), rstd


@torch.library.custom_op("kernel_opt::rms_norm_backward", mutates_args=(), device_types="cuda")
def _op_backward(h: torch.Tensor, weight: torch.Tensor, rstd: torch.Tensor, g_y: torch.Tensor,
                 g_h: torch.Tensor | None, need_w: bool) -> tuple[torch.Tensor, torch.Tensor]:
    d_x, d_w = _backward(h, weight, rstd, g_y, g_h, need_w)
    return d_x, d_w if need_w else weight.new_empty(0)


@_op_backward.register_fake
def _(h, weight, rstd, g_y, g_h, need_w):
    d_x = torch.empty(h.shape, dtype=h.dtype, device=h.device)
    return d_x, weight.new_empty(weight.shape if need_w else 0)


def _op_setup_context(ctx, inputs, output):
    x, residual, weight, _eps = inputs
    _y, h, rstd = output
    ctx.has_h = residual is not None
    ctx.save_for_backward(h if ctx.has_h else x, weight, rstd)
    ctx.mark_non_differentiable(rstd)
    ctx.set_materialize_grads(False)


def _op_backward_rule(ctx, g_y, g_h, _g_rstd):
    def backward(h, weight, rstd, g_y, g_h, need_w):
        d_x, d_w = _op_backward(h, weight, rstd, g_y, g_h, need_w)
        return d_x, d_w if need_w else None

    return *_gradients(ctx, g_y, g_h if ctx.has_h else None, backward), None


_op_forward.register_autograd(_op_backward_rule, setup_context=_op_setup_context)


def fused_rms_norm(x: torch.Tensor, weight: torch.Tensor, eps: float = 1e-6):
    """``round(x * (mean(x^2) + eps)^-1/2 * weight)`` over the last dim,
    differentiable in ``x`` and ``weight``.

    Args:
        x: ``[..., dim]`` bf16 / fp16 / fp32 on the GPU, dim at most 65536.
        weight: ``[dim]``, of ``x``'s dtype or float32.
    """
    _check(x, None, weight, eps)
    if torch.compiler.is_compiling():
        return torch.ops.kernel_opt.rms_norm(x, None, weight, float(eps))[0]
    try:
        return binding.rms_norm(x, None, weight, float(eps))[0]
    except binding.CaptureDeclined:
        return _FusedRmsNorm.apply(x, None, weight, float(eps))


def fused_add_rms_norm(x: torch.Tensor, residual: torch.Tensor, weight: torch.Tensor,
                       eps: float = 1e-6):
    """``(y, h)``: ``h = round(x + residual)``, the next residual, and its
    norm ``y`` as :func:`fused_rms_norm` gives it, differentiable in ``x``,
    ``residual`` and ``weight`` through both outputs."""
    _check(x, residual, weight, eps)
    if torch.compiler.is_compiling():
        return torch.ops.kernel_opt.rms_norm(x, residual, weight, float(eps))[:2]
    try:
        return tuple(binding.rms_norm(x, residual, weight, float(eps)))
    except binding.CaptureDeclined:
        return _FusedRmsNorm.apply(x, residual, weight, float(eps))


def fused_rms_norm_fp8(x: torch.Tensor, weight: torch.Tensor, eps: float = 1e-6):
    """``(codes, scales)`` of :func:`fused_rms_norm`'s unrounded output: e4m3
    ``[..., dim]`` and float32 ``[..., ceil(dim / 128)]``; per 128 columns with
    a = max |y|, ``scale = a / 448`` (1 where a is 0) and ``code = e4m3(y * (448
    / a))``.  A block with a NaN or an infinity stands for NaN.  No gradient:
    the outputs are detached from inputs that require one."""
    _check(x, None, weight, eps)
    try:
        return tuple(binding.rms_norm_fp8(x, None, weight, float(eps)))
    except binding.CaptureDeclined:
        pass
    return _forward(x.detach(), None, weight.detach(), eps, True)[0]


def fused_add_rms_norm_fp8(x: torch.Tensor, residual: torch.Tensor, weight: torch.Tensor,
                           eps: float = 1e-6):
    """``(codes, scales, h)``: :func:`fused_rms_norm_fp8` of ``h = round(x +
    residual)``, and ``h``.  No gradient: the outputs, ``h`` among them, are
    detached from inputs that require one."""
    _check(x, residual, weight, eps)
    try:
        return tuple(binding.rms_norm_fp8(x, residual, weight, float(eps)))
    except binding.CaptureDeclined:
        pass
    y, h, _ = _forward(x.detach(), residual.detach(), weight.detach(), eps, True)
    return y[0], y[1], h
