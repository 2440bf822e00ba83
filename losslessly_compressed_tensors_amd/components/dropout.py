"""Dropout whose mask is drawn from a counter and never stored.

The reference's trainer has none.  What backward needs of the mask is the seed
and the offset: nothing is kept between forward and backward, compressed or not.
"""
from __future__ import annotations

import math

import torch
from torch import Tensor
from torch.autograd.function import once_differentiable

from ..kernels import attention as kernels
from .attention import _check_like, _check_memory, _check_tensor, _recorded, _whole

__all__ = ["dropout_add"]

_TYPES = tuple(kernels.TYPES)


def _whole_rows(t: Tensor) -> Tensor:
    t = t.contiguous()
    return t.clone() if t.data_ptr() & 15 else t


class _DropoutAdd(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, below, seed, offset, more):
        ctx.draw = below, seed, offset
        # The device's offset may move on before backward: its own copy.
        ctx.save_for_backward(None if more is None else more.clone())
        return kernels.dropout(_whole_rows(x), None if residual is None else _whole_rows(residual),
                               below, seed, offset, more)

    @staticmethod
    def backward(ctx, grad):
        # With a graph of the backward pass asked for, a second one is an error.
        if torch.is_grad_enabled():
            return _backward_once(ctx, grad)
        return _backward(ctx, grad)


def _backward(ctx, grad):
    below, seed, offset = ctx.draw
    more, = ctx.saved_tensors
    grad_x = None
    if ctx.needs_input_grad[0]:
        grad_x = kernels.dropout(_whole_rows(grad), None, below, seed, offset, more)
    return grad_x, grad if ctx.needs_input_grad[1] else None, None, None, None, None


_backward_once = once_differentiable(_backward)


@torch.compiler.disable
def dropout_add(x: Tensor, residual: Tensor | None, p: float, seed: int, offset=0) -> Tensor:
    """``residual + dropout(x)`` of BF16, FP16 or FP32 tensors of one shape
    (``residual`` None: ``dropout(x)``), in FP32, rounded once.

    Value i (in row-major order) is dropped by 16 bits of Philox-4x32-10 at
    counter (i / 8, offset) under the key ``seed``, with ``p`` rounded to a multiple
    of 2^-16; what is kept is divided by the chance of being kept.  The same seed
    and offset give the same mask: pass another ``offset`` (or seed) for every
    layer and step.  ``seed`` and ``offset``: integers modulo 2^64; ``offset`` may be
    a one-element INT64 tensor on the device, which a captured step can advance.
    Differentiable in both; the mask is drawn again in backward."""
    _check_tensor(x, "x", x.ndim if isinstance(x, Tensor) else 0, _TYPES)
    if residual is not None:
        _check_like(residual, "residual", x, x.ndim)
        if residual.shape != x.shape:
            raise ValueError(f"x has shape {tuple(x.shape)}, residual {tuple(residual.shape)}")
    if not (math.isfinite(p) and 0 <= p <= 1):
        raise ValueError("p must lie between 0 and 1")
    seed = _whole(seed, "seed", -2 ** 63, 2 ** 64 - 1) % 2 ** 64
    more = None
    if isinstance(offset, Tensor):
        _check_memory(offset, "offset")
        if offset.dtype != torch.int64 or offset.numel() != 1 or offset.device != x.device:
            raise ValueError("an offset tensor must be one int64 on x's device")
        offset, more = 0, offset
    else:
        offset = _whole(offset, "offset", -2 ** 63, 2 ** 64 - 1) % 2 ** 64
    if x.numel() > (1 << 35) - 2048:
        raise ValueError("at most 2^35 - 2048 values")
    if x.numel() == 0:
        return x.clone() if residual is None else x + residual
    below = round(p * 65536)
    if _recorded(x, residual):
        return _DropoutAdd.apply(x, residual, below, seed, offset, more)
    return kernels.dropout(_whole_rows(x), None if residual is None else _whole_rows(residual),
                           below, seed, offset, more)
