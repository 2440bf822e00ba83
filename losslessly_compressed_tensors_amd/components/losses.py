"""Softmax cross entropy of a projection onto a large vocabulary, without its logits.

The reference's trainer projects a chunk of tokens, keeps the logits and their
gradient, and computes the capped loss in passes over both
(``examples/nanogpt/train_gpt_lct.py:88-140``).  :func:`linear_cross_entropy` computes
the loss in the projection's kernel and the logits again for the gradients, a piece
of the vocabulary at a time.  ``components/layers.py``'s ``RMSLinearCrossEntropy`` is the
training layer that keeps its input compressed.
"""
from __future__ import annotations

import math

import torch
from torch import Tensor

from ..kernels import products as kernels
from .attention import _check_like, _check_memory, _check_tensor, _recorded, _whole
from .autograd import first_order

__all__ = ["linear_cross_entropy"]

_TYPES = (torch.bfloat16, torch.float16)
_INDICES = (torch.int32, torch.int64)
REDUCTIONS = ("mean", "sum", "none")


class _LinearCrossEntropy(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, targets, softcap, ignore_index, reduction):
        out, stats = kernels.cross_entropy_forward(
            x, weight, None if bias is None else bias.float(), targets, softcap, ignore_index,
            reduction, True)
        ctx.how = softcap, ignore_index, reduction
        ctx.save_for_backward(x, weight, bias, targets, stats)
        # The caller's losses are its own to change.
        return out.clone() if reduction == "none" else out

    @staticmethod
    @first_order
    def backward(ctx, grad):
        x, weight, bias, targets, stats = ctx.saved_tensors
        grad_x, grad_weight, grad_bias = kernels.cross_entropy_backward(
            grad.contiguous(), x, weight, None if bias is None else bias.float(), targets, stats,
            *ctx.how, ctx.needs_input_grad[:3])
        if grad_bias is not None:
            grad_bias = grad_bias.to(bias.dtype)
        return grad_x, grad_weight, grad_bias, None, None, None, None


def check_cross_entropy(x, weight, targets, bias, softcap, ignore_index, reduction) -> tuple:
    """``(softcap, ignore_index)`` of checked arguments, a softcap of 0 for none."""
    if not isinstance(x, Tensor) or x.ndim < 1:
        raise TypeError("x must be a torch.Tensor of at least one dimension")
    _check_tensor(x, "x", x.ndim, _TYPES)
    _check_like(weight, "weight", x, 2)
    vocab, dim = weight.shape
    shape, device = x.shape, x.device
    if shape[-1] != dim:
        raise ValueError(f"x has {shape[-1]} channels, weight {dim}")
    if not 1 <= dim <= kernels.MAX_DIM - 7:
        raise ValueError(f"channels must lie between 1 and {kernels.MAX_DIM - 7}, got {dim}")
    if not 1 <= vocab <= kernels.MAX_VOCAB:
        raise ValueError(f"the vocabulary must lie between 1 and {kernels.MAX_VOCAB}, got {vocab}")
    _check_memory(targets, "targets")
    if targets.dtype not in _INDICES:
        raise TypeError(f"targets must be int32 or int64, got {targets.dtype}")
    if targets.shape != shape[:-1]:
        raise ValueError(f"targets must have shape {tuple(shape[:-1])}, "
                         f"got {tuple(targets.shape)}")
    if targets.device != device:
        raise ValueError(f"all tensors must be on {device}, targets is on {targets.device}")
    if targets.numel() > kernels.MAX_TOKENS:
        raise ValueError(f"at most {kernels.MAX_TOKENS} tokens")
    if targets.numel() * vocab > kernels.MAX_LOGITS:
        raise ValueError(f"tokens times vocabulary must not exceed {kernels.MAX_LOGITS}")
    if bias is not None:
        _check_tensor(bias, "bias", 1, (torch.float32, x.dtype))
        if bias.shape[0] != vocab:
            raise ValueError(f"bias must have {vocab} values, got {bias.shape[0]}")
        if bias.device != device:
            raise ValueError(f"all tensors must be on {device}, bias is on {bias.device}")
    if reduction not in REDUCTIONS:
        raise ValueError(f"reduction must be one of {', '.join(REDUCTIONS)}, got {reduction!r}")
    if softcap is None:
        softcap = 0.0
    elif not (math.isfinite(softcap) and 2.0 ** -40 <= softcap <= 2.0 ** 40):
        raise ValueError("softcap must be positive, between 2^-40 and 2^40, or None")
    return float(softcap), _whole(ignore_index, "ignore_index", -2 ** 63, 2 ** 63 - 1)


@torch.compiler.disable
def linear_cross_entropy(x: Tensor, weight: Tensor, targets: Tensor, bias: Tensor | None = None, *,
                         softcap: float | None = None, ignore_index: int = -100,
                         reduction: str = "mean") -> Tensor:
    """The cross entropy of ``softmax(l)`` with ``l = x @ weight.T + bias``, in FP32.

    ``x`` [.., channel] and ``weight`` [vocabulary, channel] are BF16 or FP16, ``bias``
    FP32 or of their type, ``targets`` [..] INT32 or INT64.  ``softcap`` s: the logits are
    ``l / sqrt(1 + (l / s)^2)``.  Tokens whose target is ``ignore_index`` have loss 0 and
    no gradients, whatever their ``x`` holds; other targets outside the vocabulary give
    NaN.  ``reduction``: "mean" over the tokens that count (0 if none does), "sum", or
    "none" for each token's loss.  Differentiable in ``x``, ``weight`` and ``bias``.

    No logits are kept: forward needs 16 bytes per token and 128 of the vocabulary
    (of up to 32 tokens: twice that), backward their gradient in 16 bits for as much of
    the vocabulary at a time as 256 MiB hold (256 words at least), 1 to 32 parts of the
    gradient of ``x`` in FP32 (the more, the fewer tokens), and of ``bias``'s gradient 8 bytes
    per 192 tokens and word.  Both directions also take a copy of ``x`` (forward of more than
    256 tokens), whether all tokens count or not, and with channels that are no multiple of 8
    widened copies of ``x``, ``weight`` and their gradients.
    Logits, softmax and sums are FP32; the logits' gradients are rounded to 16 bits for
    their products with ``weight`` and ``x`` (of up to 128 tokens, kept in two numbers)."""
    softcap, ignore_index = check_cross_entropy(x, weight, targets, bias, softcap, ignore_index,
                                                reduction)
    shape = targets.shape
    if targets.numel() == 0:
        # Nothing counts: zeros, with gradients of zero.
        zero = x.new_zeros(shape if reduction == "none" else (), dtype=torch.float32)
        if not _recorded(x, weight, bias):
            return zero
        return _Nothing.apply(zero, x, weight, bias)
    if x.ndim != 2:
        x, targets = x.reshape(-1, x.shape[-1]), targets.reshape(-1)
    targets = targets.contiguous()
    if bias is not None:
        bias = bias.contiguous()
    if _recorded(x, weight, bias):
        out = _LinearCrossEntropy.apply(x, weight, bias, targets, softcap, ignore_index, reduction)
    else:
        out, _ = kernels.cross_entropy_forward(
            x, weight, None if bias is None else bias.float(), targets, softcap, ignore_index,
            reduction, False)
    return out.view(shape) if reduction == "none" and len(shape) != 1 else out


class _Nothing(torch.autograd.Function):
    @staticmethod
    def forward(ctx, zero, *inputs):
        ctx.save_for_backward(*inputs)
        return zero.clone()

    @staticmethod
    def backward(ctx, grad):
        return None, *(torch.zeros_like(t) if t is not None and n else None
                       for t, n in zip(ctx.saved_tensors, ctx.needs_input_grad[1:]))
