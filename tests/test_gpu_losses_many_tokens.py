"""The cross entropy of a projection at the numbers of tokens that training has, against its
definition in 64 bits (``tests/product_oracle.py``): losses joined by one wave a token (more than
1024), tokens listed in several rounds (more than 16384), several pieces of the vocabulary, and
tokens that do not count at each of them."""
from __future__ import annotations

import pytest
import torch

from gpu_util import require_gpu
from losslessly_compressed_tensors_amd.components.losses import linear_cross_entropy
from losslessly_compressed_tensors_amd.kernels import products
from product_oracle import CrossEntropy, assert_within
from test_gpu_losses import _check, _inputs

pytestmark = pytest.mark.gpu
BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32


@pytest.fixture(autouse=True)
def _gpu():
    require_gpu()


def _grad(tokens, reduction):
    if reduction != "none":
        return None
    return torch.randn(tokens, generator=torch.Generator().manual_seed(1))


@pytest.mark.parametrize("reduction", ["mean", "none"])
@pytest.mark.parametrize("ignored", [0.0, 0.3])
@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("tokens,vocab,dim", [(1024, 130, 16), (1025, 300, 24), (1027, 555, 40),
                                              (2050, 300, 24)])
def test_one_wave_a_token(tokens, vocab, dim, dtype, ignored, reduction):
    x, weight, targets, bias = _inputs(tokens, vocab, dim, dtype, bias=FP32, ignored=ignored)
    _check(x, weight, targets, bias, reduction=reduction, grad=_grad(tokens, reduction))


@pytest.mark.parametrize("softcap", [None, 15.0])
def test_parts_of_many_tiles_of_the_vocabulary(softcap):
    x, weight, targets, bias = _inputs(1100, 40000, 16, BF16, bias=FP32, ignored=0.1)
    _check(x, weight, targets, bias, softcap=softcap)


# 16384 tokens a round.
@pytest.mark.parametrize("reduction", ["mean", "none"])
@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("tokens", [16384, 16385, 33000])
def test_tokens_are_listed_in_rounds(tokens, dtype, reduction):
    x, weight, targets, bias = _inputs(tokens, 20, 8, dtype, bias=FP32, ignored=0.2)
    for border in (16384, 32768):
        targets[border - 3:border + 2] = torch.tensor([-100, 3, -100, -100, 7])[:len(
            targets[border - 3:border + 2])]
    _check(x, weight, targets, bias, reduction=reduction, grad=_grad(tokens, reduction))


@pytest.mark.parametrize("kept", ["first", "last", "none"])
def test_rounds_of_which_all_or_none_count(kept):
    tokens = 33000
    x, weight, targets, bias = _inputs(tokens, 20, 8, BF16, bias=FP32)
    if kept == "first":
        targets[16384:] = -100
    elif kept == "last":
        targets[:32768] = -100
    else:
        targets[:] = -100
    dirty = x.clone()
    dirty[targets == -100] = float("nan")
    plain, out = (_check(t, weight, targets, bias, reduction="sum") for t in (x, dirty))
    assert torch.equal(plain[0], out[0]) and all(map(torch.equal, plain[1], out[1]))


@pytest.mark.parametrize("reduction", ["mean", "none"])
@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("tokens", [300, 600])
def test_deep_products_of_tokens_that_count(tokens, dtype, reduction):
    x, weight, targets, bias = _inputs(tokens, 513, 2048, dtype, bias=FP32, ignored=0.3)
    _check(x, weight, targets, bias, softcap=30.0, reduction=reduction,
           grad=_grad(tokens, reduction))


def test_small_vocabularies_against_many_tokens():
    x, weight, targets, bias = _inputs(5003, 700, 72, BF16, bias=FP32, ignored=0.1)
    _check(x, weight, targets, bias, softcap=15.0)


@pytest.mark.parametrize("ignored", [0.0, 0.2])
def test_a_trainers_size(ignored):
    """Two pieces of the vocabulary and 16 tiles of tokens (the oracle's sums on the GPU, in 64
    bits too)."""
    tokens, vocab, dim = 4096, 50304, 256
    assert products.vocabulary_pieces(tokens, vocab, dim)[0] < vocab
    x, weight, targets, bias = (t.cuda() for t in _inputs(tokens, vocab, dim, BF16, bias=FP32,
                                                          ignored=ignored))
    leaves = [t.requires_grad_() for t in (x, weight, bias)]
    out = linear_cross_entropy(x, weight, targets, bias, softcap=15.0)
    grads = torch.autograd.grad(out, leaves)
    with torch.no_grad():
        exact = CrossEntropy(x, weight, targets, bias, 15.0)
    assert_within(out, exact.total.cpu(), exact.total_off.cpu(), "total")
    for name, got in zip(("grad_x", "grad_weight", "grad_bias"), grads):
        assert_within(got, getattr(exact, name).cpu(), getattr(exact, name + "_off").cpu(), name)


def _backward_peak(tokens, vocab, dim):
    x = torch.randn(tokens, dim, device="cuda").to(BF16).requires_grad_()
    weight = torch.randn(vocab, dim, device="cuda").to(BF16).requires_grad_()
    bias = torch.zeros(vocab, device="cuda", requires_grad=True)
    loss = linear_cross_entropy(x, weight, torch.zeros(tokens, dtype=torch.int64, device="cuda"),
                                bias, reduction="sum")
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    grads = torch.autograd.grad(loss, (x, weight, bias))
    return (torch.cuda.max_memory_allocated() - before
            - sum(g.numel() * g.element_size() for g in grads))


@pytest.mark.parametrize("tokens,vocab,dim", [(1, (1 << 22) + 5, 8), (128, (1 << 21) + 5, 8),
                                              (24000, 30000, 16), (4096, 50304, 256)])
def test_memory_as_stated(tokens, vocab, dim):
    piece, splits = products.vocabulary_pieces(tokens, vocab, dim)
    stated = (2 * tokens * dim                          # the counted tokens' x
              + (256 << 20) + 512 * (tokens + 7)        # the logits' gradients: a tile more
              + 4 * splits * tokens * dim               # parts of grad_x
              + 8 * -(-tokens // 192) * vocab           # of the bias's gradient
              + 20 * tokens + 8)                        # lists
    assert splits <= 32
    assert _backward_peak(tokens, vocab, dim) <= stated + (1 << 20)     # (alignment)
