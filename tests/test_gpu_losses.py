"""The cross entropy of a projection onto a vocabulary on the GPU, against its
definition in 64 bits (``tests/product_oracle.py``)."""
from __future__ import annotations

import pytest
import torch

from gpu_util import require_gpu
from losslessly_compressed_tensors_amd.components.losses import linear_cross_entropy
from product_oracle import CrossEntropy, assert_within

pytestmark = pytest.mark.gpu
BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32


@pytest.fixture(autouse=True)
def _gpu():
    require_gpu()


def _inputs(tokens, vocab, dim, dtype, bias=None, ignored=0.0, seed=0, index=torch.int64,
            spread=2.0):
    g = torch.Generator().manual_seed(seed)
    weight = torch.randn(vocab, dim, generator=g) * (spread / dim ** 0.5)
    targets = torch.randint(0, vocab, (tokens,), generator=g)
    x = torch.randn(tokens, dim, generator=g)
    x[::2] += 3 * weight[targets[::2]]
    drop = torch.rand(tokens, generator=g) < ignored
    targets[drop] = -100
    b = None if bias is None else (0.5 * torch.randn(vocab, generator=g)).to(bias)
    return x.to(dtype), weight.to(dtype), targets.to(index), b


def _check(x, weight, targets, bias=None, reduction="mean", grad=None, **how):
    """Forward and gradients of one call against the oracle; returns what it gave."""
    exact = CrossEntropy(x.cpu(), weight.cpu(), targets.cpu(), None if bias is None else bias.cpu(),
                         reduction=reduction, grad=grad, **how)
    leaves = [t.detach().cuda().requires_grad_() for t in (x, weight) + (() if bias is None
                                                                         else (bias,))]
    out = linear_cross_entropy(leaves[0], leaves[1], targets.cuda(), *leaves[2:],
                               reduction=reduction, **how)
    assert out.dtype == FP32
    if reduction == "none":
        assert out.shape == targets.shape
        assert_within(out, exact.losses, exact.losses_off, "losses")
    else:
        assert out.shape == ()
        assert_within(out, exact.total, exact.total_off, "total")
    out.backward(None if grad is None else grad.cuda())
    assert_within(leaves[0].grad, exact.grad_x, exact.grad_x_off, "grad_x")
    assert_within(leaves[1].grad, exact.grad_weight, exact.grad_weight_off, "grad_weight")
    for leaf in leaves:
        assert leaf.grad.dtype == leaf.dtype and leaf.grad.shape == leaf.shape
    if bias is not None and bias.dtype == FP32:
        assert_within(leaves[2].grad, exact.grad_bias, exact.grad_bias_off, "grad_bias")
    return out.detach(), [leaf.grad for leaf in leaves]


SIZES = [(1, 1, 8), (1, 50, 8), (3, 256, 32), (5, 257, 40), (37, 307, 72), (128, 128, 64),
         (129, 255, 96), (255, 513, 104), (257, 1000, 128), (300, 2049, 264), (64, 4096, 256),
         (520, 777, 512)]


@pytest.mark.parametrize("softcap", [None, 15.0])
@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("tokens,vocab,dim", SIZES)
def test_sizes(tokens, vocab, dim, dtype, softcap):
    x, weight, targets, bias = _inputs(tokens, vocab, dim, dtype, bias=FP32)
    _check(x, weight, targets, bias if softcap else None, softcap=softcap)


@pytest.mark.parametrize("dim", [1, 2, 7, 13, 33, 70, 129])
def test_odd_channels(dim):
    x, weight, targets, bias = _inputs(21, 67, dim, BF16, bias=FP32)
    _check(x, weight, targets, bias, reduction="sum")


@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
@pytest.mark.parametrize("ignored", [0.0, 0.4, 1.0])
@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_reductions_and_ignored_tokens(reduction, ignored, dtype):
    x, weight, targets, bias = _inputs(300, 555, 64, dtype, bias=FP32, ignored=ignored,
                                       index=torch.int32)
    grad = None
    if reduction == "none":
        grad = torch.randn(300, generator=torch.Generator().manual_seed(1)) * 1e-3
    _check(x, weight, targets, bias, reduction=reduction, grad=grad)


@pytest.mark.parametrize("scale", [1e-12, 1e-4, 1.0, 1e8])
@pytest.mark.parametrize("reduction", ["sum", "none"])
def test_incoming_gradients_of_any_size(scale, reduction):
    x, weight, targets, bias = _inputs(70, 300, 64, BF16, bias=FP32)
    grad = torch.tensor(scale)
    if reduction == "none":
        grad = scale * torch.rand(70, generator=torch.Generator().manual_seed(2))
        grad[5] = 0.0
    _check(x, weight, targets, bias, reduction=reduction, grad=grad)
