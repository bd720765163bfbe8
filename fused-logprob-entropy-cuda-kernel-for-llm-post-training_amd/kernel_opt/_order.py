"""Refusal of second derivatives through an operator whose gradients come from a kernel."""
from __future__ import annotations

import torch


class _FirstOrder(torch.autograd.Function):
    """``grads`` as functions of what they depend on, whose own gradient is
    refused: left without a graph they would count as constants in a second
    derivative."""

    @staticmethod
    def forward(ctx, name, n, *tensors):
        ctx.name = name
        return tensors[:n]

    @staticmethod
    def backward(ctx, *grads):
        raise RuntimeError(f"kernel_opt: {ctx.name} has no second derivative")


def first_order(name, grads, of):
    """The gradients ``grads`` (None where there is none) of the operator
    ``name``, refusing to be differentiated with respect to the tensors ``of``
    under ``create_graph``."""
    if not torch.is_grad_enabled():
        return grads
    given = [g for g in grads if g is not None]
    held = iter(_FirstOrder.apply(name, len(given), *given, *(t for t in of if t is not None)))
    return tuple(None if g is None else next(held) for g in grads)
