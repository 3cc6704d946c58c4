"""Gradients that have no derivative of their own say so, on the host."""
import pytest
import torch
from torch.autograd import Function, forward_ad

from fastmd_b200._first_order import first_order, has_tangent


class Square(Function):
    """x^2 with a gradient that autograd does not see into."""

    @staticmethod
    def forward(ctx, x):
        ctx.save_for_backward(x)
        return x * x

    @staticmethod
    def backward(ctx, g):
        (x,) = ctx.saved_tensors
        with torch.no_grad():
            dx = 2 * x * g
        return first_order("square", (dx, None), (g, x))[0]


def test_a_second_derivative_raises_and_a_first_one_is_as_it_was():
    x = torch.tensor([3.0, -1.0], requires_grad=True)
    (want,) = torch.autograd.grad(Square.apply(x).sum(), x)
    assert torch.equal(want, 2 * x.detach()) and not want.requires_grad
    (dx,) = torch.autograd.grad(Square.apply(x).sum(), x, create_graph=True)
    assert torch.equal(dx, want)
    with pytest.raises(RuntimeError, match="square has first derivatives only"):
        torch.autograd.grad(dx.sum() + x.sum(), x)


def test_gradients_of_constants_need_no_node():
    y = torch.tensor([2.0])
    assert first_order("constant", (y, None), (y, None)) == (y, None)


def test_what_does_not_pass_through_it_is_free():
    x, w = torch.tensor([3.0], requires_grad=True), torch.tensor([2.0], requires_grad=True)
    (dx,) = torch.autograd.grad(Square.apply(x).sum(), x, create_graph=True)
    (dw,) = torch.autograd.grad((dx * w).sum(), w)
    assert torch.equal(dw, dx.detach())


def test_a_tangent_is_seen():
    x = torch.tensor([3.0])
    assert not has_tangent(x, None)
    with forward_ad.dual_level():
        assert not has_tangent(x, None)
        dual = forward_ad.make_dual(x, torch.ones(1))
        assert has_tangent(None, x, dual)
        with pytest.raises(RuntimeError):  # an autograd function without a forward-mode rule refuses it
            Square.apply(dual)
