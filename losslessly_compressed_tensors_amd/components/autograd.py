"""What the package's autograd functions share."""
from __future__ import annotations

import functools

import torch
from torch import Tensor

__all__ = ["first_order"]


class _Constant(torch.autograd.Function):
    """A gradient whose own derivative is an error."""

    @staticmethod
    def forward(ctx, grad):
        return grad.view_as(grad)

    @staticmethod
    def backward(ctx, grad):
        raise RuntimeError("this operator can be differentiated once only: its gradients have no "
                           "derivatives")


def first_order(backward):
    """A function's ``backward`` whose gradients autograd cannot differentiate (kernels
    computed them, or what they depend on was not saved by autograd).  Where a graph
    of them is asked for (``create_graph=True``), they are the same, and a derivative of
    them is an error: without one they would pass for constants.
    (``torch.autograd.function.once_differentiable`` lets that happen where the incoming
    gradient is a constant, as at a loss.)"""

    @functools.wraps(backward)
    def run(ctx, *grads):
        if not torch.is_grad_enabled():
            return backward(ctx, *grads)
        with torch.no_grad():
            results = backward(ctx, *grads)
        if not isinstance(results, tuple):
            results = (results,)
        return tuple(_Constant.apply(t.detach().requires_grad_()) if isinstance(t, Tensor) else t
                     for t in results)

    return run
