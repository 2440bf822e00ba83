"""Dropout with the residual's addition against its definition: the generator's
words on the host, the sum in 64 bits."""
from __future__ import annotations

import attention_oracle as oracle
import pytest
import torch

from losslessly_compressed_tensors_amd.components.dropout import dropout_add

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _values(*shape, dtype=torch.bfloat16, seed=0):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(dtype).to(DEV)


def _expected(x, residual, p, seed, offset):
    keep = oracle.kept(x.numel(), p, seed, offset).view(x.shape)
    below = round(p * 65536)
    factor = 65536 / (65536 - below) if below < 65536 else 0.0
    out = torch.where(keep, x.detach().cpu().double() * factor, 0.0)
    size = out.abs()
    if residual is not None:
        out, size = out + residual.cpu().double(), size + residual.cpu().double().abs()
    # The factor and the fused product-and-sum in FP32, one rounding.
    return out, 3 * oracle.STEP * size + oracle.UNIT[x.dtype] * out.abs() + oracle.LEAST[x.dtype]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("shape", [(1,), (7,), (8,), (3, 5, 7), (2047,), (129, 768)])
@pytest.mark.parametrize("p,seed,offset", [(0.1, 0, 0), (0.5, 2 ** 64 - 1, 2 ** 63 + 5), (0.0, 3, 1),
                                           (1.0, 3, 1), (0.999, 1 << 40, 1 << 33)])
def test_dropout_and_gradient(shape, dtype, p, seed, offset):
    x, grad = _values(*shape, dtype=dtype).requires_grad_(), _values(*shape, dtype=dtype, seed=2)
    residual = _values(*shape, dtype=dtype, seed=1).requires_grad_()
    out = dropout_add(x, residual, p, seed, offset)
    exact, bound = _expected(x, residual.detach(), p, seed, offset)
    assert bool(((out.detach().cpu().double() - exact).abs() <= bound).all())
    gx, gr = torch.autograd.grad(out, (x, residual), grad)
    exact, bound = _expected(grad, None, p, seed, offset)
    assert bool(((gx.cpu().double() - exact).abs() <= bound).all())
    assert torch.equal(gr, grad)
    bare = dropout_add(x.detach(), None, p, seed, offset)
    exact, bound = _expected(x, None, p, seed, offset)
    assert bool(((bare.cpu().double() - exact).abs() <= bound).all())


def test_gradient_against_differences():
    """Linear in x: a difference of any step is the gradient."""
    x, grad = _values(4000, dtype=torch.float32), _values(4000, dtype=torch.float32, seed=1)
    leaf = x.clone().requires_grad_()
    g, = torch.autograd.grad(dropout_add(leaf, None, 0.25, 9, 4), leaf, grad)
    ahead, behind = (dropout_add(x + s * 0.5, None, 0.25, 9, 4).double() for s in (1, -1))
    assert bool(((ahead - behind) * grad.double() - g.double()).abs().amax() <= 1e-5)


def test_large_indices_and_statistics():
    """The last values of 2^27 + 5, and the share that is kept."""
    n = (1 << 27) + 5
    x = torch.ones(n, dtype=torch.bfloat16, device=DEV)
    out = dropout_add(x, None, 0.3, 77, 12)
    below = round(0.3 * 65536)
    share = float((out != 0).double().mean())
    assert abs(share - (1 - below / 65536)) < 6 * (0.25 / n) ** 0.5
    first = (n - 1000) // 8
    words = oracle.philox_words(n // 8 + 1, 77, 12)[first:]
    halves = torch.from_numpy(words.copy().view("<u2").reshape(-1)[:n - 8 * first] >= below)
    assert torch.equal((out[8 * first:] != 0).cpu(), halves)


def test_the_generator_is_the_published_one():
    """Philox-4x32-10's published answer for counter 0 and key 0."""
    words = oracle.philox_words(1, 0, 0)[0]
    assert [int(w) for w in words] == [0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8]


def test_dropped_infinities_and_nans_are_gone():
    x = torch.full((4096,), float("inf"), device=DEV)
    x[::2] = float("nan")
    residual = _values(4096, dtype=torch.float32)
    keep = oracle.kept(4096, 0.5, 5, 0).to(DEV)
    out = dropout_add(x, residual, 0.5, 5)
    assert torch.equal(out[~keep], residual[~keep])
    assert not bool(out[keep].isfinite().any())


def test_an_offset_on_the_device_and_strided_inputs():
    x, residual = _values(64, 96).t(), _values(96, 64, seed=1)
    want = dropout_add(x.contiguous(), residual, 0.4, 11, 6)
    offset = torch.tensor([6], device=DEV)
    leaf = x.detach().requires_grad_()
    out = dropout_add(leaf, residual, 0.4, 11, offset)
    assert torch.equal(out, want)
    offset += 1                                   # the mask of backward stays the forward's
    g, = torch.autograd.grad(out, leaf, torch.ones_like(out))
    keep = oracle.kept(96 * 64, 0.4, 11, 6).view(96, 64).to(DEV)
    assert torch.equal(g != 0, keep)
    odd = torch.zeros(1001, dtype=torch.bfloat16, device=DEV)[1:]
    odd.copy_(_values(1000))
    assert torch.equal(dropout_add(odd, None, 0.4, 2), dropout_add(_values(1000), None, 0.4, 2))
    empty = _values(0, 5)
    assert dropout_add(empty, empty, 0.1, 1).shape == (0, 5)


def test_refusals():
    x = _values(4, 8)
    for bad, error, match in (
            (lambda: dropout_add(x.cpu(), None, 0.1, 1), ValueError, "GPU"),
            (lambda: dropout_add(x.double(), None, 0.1, 1), TypeError, "bfloat16"),
            (lambda: dropout_add(x, x.float(), 0.1, 1), TypeError, "one type"),
            (lambda: dropout_add(x, x[:3], 0.1, 1), ValueError, "shape"),
            (lambda: dropout_add(x, None, 1.5, 1), ValueError, "p must"),
            (lambda: dropout_add(x, None, float("nan"), 1), ValueError, "p must"),
            (lambda: dropout_add(x, None, 0.1, 1.0), TypeError, "seed"),
            (lambda: dropout_add(x, None, 0.1, 2 ** 64), ValueError, "seed"),
            (lambda: dropout_add(x, None, 0.1, 1, torch.zeros(2, device=DEV)), ValueError,
             "offset"),
            (lambda: dropout_add(None, None, 0.1, 1), TypeError, "Tensor")):
        with pytest.raises(error, match=match):
            bad()
