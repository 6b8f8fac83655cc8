"""What the operators' autograd functions share."""
from __future__ import annotations

import torch
from torch import Tensor
from torch.autograd import Function, forward_ad


class _FirstOnly(Function):
    """Gradients as they are; differentiating them raises."""

    @staticmethod
    def forward(ctx, name: str, count: int, *tensors):
        ctx.name = name
        return tuple(None if x is None else x.view_as(x) for x in tensors[:count])

    @staticmethod
    def backward(ctx, *grads):
        raise NotImplementedError(f"{ctx.name} has first derivatives only: its gradients cannot be differentiated again")


def first_derivatives(name: str, grads: tuple, *inputs: Tensor | None) -> tuple:
    """``grads`` for a backward that is not itself differentiable. Under ``create_graph`` they depend on ``inputs`` (the
    gradients that came in and the forward's own inputs) through a function that raises, where kernels alone would leave
    constants and their part of a second derivative would be missing without a word."""
    if not torch.is_grad_enabled() or not any(x is not None and x.requires_grad for x in inputs):
        return grads
    return _FirstOnly.apply(name, len(grads), *grads, *inputs)


def differentiated(*tensors: Tensor | None) -> bool:
    """Whether a call on these tensors belongs to autograd: gradients are wanted, or one of them carries a tangent (for which
    an autograd function without a forward-mode rule raises)."""
    if torch.is_grad_enabled() and any(x is not None and x.requires_grad for x in tensors):
        return True
    if forward_ad._current_level < 0:  # outside every dual level, as nearly always
        return False
    return any(x is not None and forward_ad.unpack_dual(x).tangent is not None for x in tensors)
