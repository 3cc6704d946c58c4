"""Operators whose gradients are filled in by kernels have first derivatives only; this says so where more is asked."""
from __future__ import annotations

import torch
from torch.autograd import Function, forward_ad


class _Refuse(Function):
    """The gradients as they are; to differentiate them raises."""

    @staticmethod
    def forward(ctx, name, count, *tensors):
        ctx.name = name
        return tuple(t.detach() for t in tensors[:count])

    @staticmethod
    def backward(ctx, *grads):
        raise RuntimeError(f"{ctx.name} has first derivatives only: its gradient cannot be differentiated")


def first_order(name: str, grads, inputs) -> tuple:
    """``grads`` (None: none) of operator ``name``, which depend on ``inputs``. Where autograd records the backward pass
    (``create_graph``) and an input requires a gradient, a second derivative raises: without a node of its own a gradient
    is a constant to autograd, which would drop the term without a word."""
    if not torch.is_grad_enabled():
        return tuple(grads)
    some = [g for g in grads if g is not None]
    kept = iter(_Refuse.apply(name, len(some), *some, *(t for t in inputs if t is not None)))
    return tuple(None if g is None else next(kept) for g in grads)


def has_tangent(*tensors) -> bool:
    """Whether one of the tensors (None: none) carries a tangent of forward mode. Such a call goes through the operator's
    autograd function, which refuses it; a call past it would lose the tangent."""
    if getattr(forward_ad, "_current_level", 0) < 0:  # outside forward mode, at the cost of a look (else 0.4 us a tensor)
        return False
    return any(t is not None and forward_ad.unpack_dual(t).tangent is not None for t in tensors)
