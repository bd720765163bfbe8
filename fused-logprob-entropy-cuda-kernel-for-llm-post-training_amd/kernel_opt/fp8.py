"""8-bit (e4m3) matrices with a float32 scale per block of 128: quantization
and the product of an LM head on them.

A block of values v with a = max |v| is held as ``code = e4m3(v * (448 / a))``
and ``scale = a / 448`` (1 where a is 0), and stands for ``code * scale``.
Activations share a scale over 128 columns of a row, weights over 128 x 128
elements; :func:`kernel_opt.fused_add_rms_norm_fp8` writes the former.

``fp8_linear(x, x_scale, weight, weight_scale)`` is their product ``[..., N]``
(csrc/klp_fp8_gemm.hip): each 128 of the inner dim is one matrix instruction
on the codes, whose float32 sums are scaled and added in float32.  For a 16-bit
``out_dtype`` that is the e4m3 instruction, which cuts products more than 13
bits below the largest of 8 neighbours (5 10^-5 of a result on normal data, a
hundredth of the output's rounding); for float32 the bf16 one, with exact
products, at about half the rate.  There is no gradient: codes are data, not
leaves.
"""
from __future__ import annotations

import torch

from ._library import (DTYPE_CODES, binding, check_status, device_guard, lib, ptr,
                       stream_handle)
from .norm import SCALE_BLOCK, _rows

__all__ = ["quantize_fp8", "fp8_linear"]

MAX_ROWS = 2 ** 20  # of one product's x


def quantize_fp8(x: torch.Tensor, block_rows: int = 1):
    """``(codes, scales)`` of ``x`` ``[..., dim]`` (bf16 / fp16 / fp32, GPU).

    ``block_rows=1``: scales ``[..., ceil(dim / 128)]``, 128 columns of a row
    each.  ``block_rows=128`` (a weight ``[N, dim]``): scales ``[ceil(N / 128),
    ceil(dim / 128)]``, 128 x 128 elements each.  A block with a NaN or an
    infinity stands for NaN.  No gradient: the outputs are detached from an
    ``x`` that requires one.
    """
    if not x.is_cuda:
        raise RuntimeError("x must be a GPU tensor")
    if x.dtype not in DTYPE_CODES:
        raise RuntimeError("x must be bf16, fp16, or fp32")
    if block_rows not in (1, SCALE_BLOCK):
        raise ValueError(f"block_rows must be 1 or {SCALE_BLOCK}, got {block_rows}")
    if x.dim() < 1 or x.size(-1) < 1 or (block_rows != 1 and x.dim() != 2):
        raise RuntimeError(f"x must be {'[..., dim]' if block_rows == 1 else '[N, dim]'} with "
                           f"dim >= 1, got {tuple(x.shape)}")
    try:
        return tuple(binding.quantize_fp8(x, int(block_rows)))
    except binding.CaptureDeclined:
        x = x.detach()
    dev = x.device
    D = x.size(-1)
    nb = -(-D // SCALE_BLOCK)
    x2, ld = _rows(x)
    N = x2.size(0)
    q = torch.empty(x.shape, dtype=torch.float8_e4m3fn, device=dev)
    lead = x.shape[:-1] if block_rows == 1 else (-(-N // SCALE_BLOCK),)
    scales = torch.empty(*lead, nb, dtype=torch.float32, device=dev)
    with device_guard(dev.index):
        check_status(lib.klp_quantize_fp8(ptr(x2), DTYPE_CODES[x.dtype], ld, N, D, int(block_rows),
                                          ptr(q), ptr(scales), stream_handle(dev.index)))
    return q, scales


def _check_linear(x, x_scale, weight, weight_scale, out_dtype):
    named = (("x", x), ("x_scale", x_scale), ("weight", weight), ("weight_scale", weight_scale))
    if not all(t.is_cuda for _, t in named):
        raise RuntimeError("x, weight and their scales must be GPU tensors")
    if any(t.device != x.device for _, t in named):
        raise RuntimeError("x, weight and their scales must be on the same device")
    if x.dtype != torch.float8_e4m3fn or weight.dtype != torch.float8_e4m3fn:
        raise RuntimeError("x and weight must be float8_e4m3fn")
    if x_scale.dtype != torch.float32 or weight_scale.dtype != torch.float32:
        raise RuntimeError("scales must be float32")
    if out_dtype not in DTYPE_CODES:
        raise RuntimeError("out_dtype must be bf16, fp16, or fp32")
    if x.dim() < 1 or weight.dim() != 2 or weight.size(0) < 1 or weight.size(1) != x.size(-1):
        raise RuntimeError(f"x must be [..., K] and weight [N, K], got {tuple(x.shape)} and "
                           f"{tuple(weight.shape)}")
    N, K = weight.shape
    if K < 16 or K % 16:
        raise RuntimeError(f"K must be a positive multiple of 16, got {K}")
    nb = -(-K // SCALE_BLOCK)
    if tuple(x_scale.shape) != (*x.shape[:-1], nb):
        raise RuntimeError(f"x_scale must be {(*x.shape[:-1], nb)}, got {tuple(x_scale.shape)}")
    if tuple(weight_scale.shape) != (-(-N // SCALE_BLOCK), nb):
        raise RuntimeError(f"weight_scale must be {(-(-N // SCALE_BLOCK), nb)}, got "
                           f"{tuple(weight_scale.shape)}")
    if torch.is_grad_enabled() and any(t.requires_grad for _, t in named):
        raise RuntimeError("fp8_linear has no gradient: pass detached codes and scales")


def fp8_linear(x: torch.Tensor, x_scale: torch.Tensor, weight: torch.Tensor,
               weight_scale: torch.Tensor, out_dtype: torch.dtype = torch.bfloat16):
    """``out[..., n] = sum_k x[..., k] x_scale[..., k / 128] * weight[n, k]
    weight_scale[n / 128, k / 128]``, float32 sums rounded once to
    ``out_dtype``.

    Args:
        x: ``[..., K]`` float8_e4m3fn, K a multiple of 16, at most 2**20 rows.
        x_scale: ``[..., ceil(K / 128)]`` float32.
        weight: ``[N, K]`` float8_e4m3fn.
        weight_scale: ``[ceil(N / 128), ceil(K / 128)]`` float32.

    Rows of ``x`` and ``weight`` start at multiples of 16 bytes (RuntimeError
    otherwise).  A NaN code or scale gives NaN in the outputs it enters.  The
    two scales of a block are multiplied first, in float32: their product has
    to stay in its range.
    """
    _check_linear(x, x_scale, weight, weight_scale, out_dtype)
    try:
        return binding.fp8_linear(x, x_scale, weight, weight_scale, out_dtype)
    except binding.CaptureDeclined:
        pass
    dev = x.device
    x2, ld_x = _rows(x)
    w2, ld_w = _rows(weight)
    xs, ws = x_scale.contiguous(), weight_scale.contiguous()
    M, N, K = x2.size(0), w2.size(0), w2.size(1)
    out = torch.empty(*x.shape[:-1], N, dtype=out_dtype, device=dev)
    with device_guard(dev.index):
        check_status(lib.klp_fp8_linear(ptr(x2), ld_x, ptr(xs), ptr(w2), ld_w, ptr(ws), M, N, K,
                                        DTYPE_CODES[out_dtype], ptr(out), N,
                                        stream_handle(dev.index)))
    return out
