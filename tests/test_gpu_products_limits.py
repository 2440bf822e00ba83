"""The product operators at the ends of what they take: the most tokens, words, channels and
columns; odd channels in captured steps; two streams at once; memory that holds anything."""
from __future__ import annotations

import math

import pytest
import torch

from gpu_util import require_gpu
from losslessly_compressed_tensors_amd.components.losses import linear_cross_entropy
from losslessly_compressed_tensors_amd.components.orthogonal import orthogonalize
from product_oracle import CrossEntropy, assert_within, polar, polar_off
from test_gpu_losses import _check, _inputs
from test_gpu_orthogonal import _matrix

pytestmark = pytest.mark.gpu
BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32


@pytest.fixture(autouse=True)
def _gpu():
    require_gpu()


def test_most_tokens():
    x, weight, targets, bias = (t.cuda() for t in _inputs(1 << 22, 5, 8, BF16, bias=FP32,
                                                          ignored=0.1))
    leaves = [t.requires_grad_() for t in (x, weight, bias)]
    out = linear_cross_entropy(x, weight, targets, bias)
    grads = torch.autograd.grad(out, leaves)
    with torch.no_grad():
        exact = CrossEntropy(x, weight, targets, bias)
    assert_within(out, exact.total.cpu(), exact.total_off.cpu(), "total")
    for name, got in zip(("grad_x", "grad_weight", "grad_bias"), grads):
        assert_within(got, getattr(exact, name).cpu(), getattr(exact, name + "_off").cpu(), name)


@pytest.mark.parametrize("tokens", [3, 150])
def test_most_words(tokens):
    x, weight, targets, _ = (t if t is None else t.cuda()
                             for t in _inputs(tokens, 1 << 24, 8, BF16))
    targets[:2] = torch.tensor([0, (1 << 24) - 1])
    leaves = [t.requires_grad_() for t in (x, weight)]
    out = linear_cross_entropy(x, weight, targets, reduction="sum")
    grads = torch.autograd.grad(out, leaves)
    lse, grad_x = [], []
    with torch.no_grad():
        w, sums = weight.double(), []
        for n in range(tokens):
            z = (w * x[n].double()).sum(1)
            sums.append(torch.logsumexp(z, 0))
            lse.append(sums[-1] - z[targets[n]])
            p = torch.softmax(z, 0)
            p[targets[n]] -= 1
            if n < 3:
                grad_x.append(((p[:, None] * w).sum(0), (p[:, None] * w).abs().sum(0)))
        exact = torch.stack(lse).sum()
        # FP32 sums of 8 products and a maximum, of logits below 64; sums of 2^24 exponentials.
        assert abs(float(out.detach()) - float(exact)) <= 1e-4 * float(exact)
        for n, (gx, size) in enumerate(grad_x):
            # dz and the result in BF16, FP32 sums of up to 2^24 products.
            off = (2.0 ** -8 + 2.0 ** -14) * size + 2.0 ** -8 * gx.abs()
            assert_within(grads[0][n], gx.cpu(), (1.01 * off).cpu(), "grad_x")
        # Words that are no target and all the targets', over the tokens.
        rows = torch.cat([targets.unique(), torch.arange(100, 100000, 997, device="cuda")])
        z = x.double() @ w[rows].T
        p = (z - torch.stack(sums)[:, None]).exp()
        p -= (targets[:, None] == rows).double()
        gw, size = p.T @ x.double(), p.abs().T @ x.double().abs()
        off = (2.0 ** -8 + 2.0 ** -14) * size + 2.0 ** -8 * gw.abs()
        assert_within(grads[1][rows], gw.cpu(), (1.01 * off + 1e-30).cpu(), "grad_weight")


def test_most_logits():
    """2^37 of them, in 1024 pieces: zero weights, so each probability is 2^-24."""
    tokens, vocab, dim = 1 << 13, 1 << 24, 8
    g = torch.Generator(device="cuda").manual_seed(0)
    x = torch.randn(tokens, dim, generator=g, device="cuda").to(BF16).requires_grad_()
    weight = torch.zeros(vocab, dim, dtype=BF16, device="cuda", requires_grad=True)
    targets = torch.randint(0, vocab, (tokens,), generator=g, device="cuda")
    out = linear_cross_entropy(x, weight, targets)
    assert abs(float(out.detach()) - 24 * math.log(2)) < 1e-5
    grads = torch.autograd.grad(out, (x, weight))
    assert not grads[0].any()
    exact = (x.detach().double().sum(0) * 2.0 ** -24).repeat(vocab, 1)
    size = (x.detach().double().abs().sum(0) * 2.0 ** -24).repeat(vocab, 1)
    exact.index_add_(0, targets, -x.detach().double())
    size.index_add_(0, targets, x.detach().double().abs())
    off = 2.0 ** -8 * exact.abs() + (2.0 ** -8 + tokens * 2.0 ** -24) * size
    assert ((grads[1].double() * tokens - exact).abs() <= 1.01 * off).all()


@pytest.mark.parametrize("tokens", [5, 300])
@pytest.mark.parametrize("dim", [65528, 65529])
def test_most_channels(dim, tokens):
    x, weight, targets, bias = _inputs(tokens, 270, dim, BF16, bias=FP32, ignored=0.2)
    _check(x, weight, targets, bias, reduction="sum")


@pytest.mark.parametrize("tokens", [3, 300])
def test_longest_rows(tokens):
    """Rows at a stride that the kernels take, and past it."""
    x, weight, targets, bias = (t.cuda() for t in _inputs(tokens, 270, 64, BF16, bias=FP32))
    base = linear_cross_entropy(x, weight, targets, bias)
    for stride in (65536, 65544):
        wide = [torch.full((len(t), stride), float("nan"), dtype=BF16, device="cuda")
                for t in (x, weight)]
        for to, t in zip(wide, (x, weight)):
            to[:, :64] = t
        assert torch.equal(linear_cross_entropy(wide[0][:, :64], wide[1][:, :64], targets, bias),
                           base)


@pytest.mark.parametrize("shape", [(3, 65536), (65536, 5), (70, 65536), (65535, 130)])
def test_longest_matrices(shape):
    g = _matrix(shape).to(BF16)
    exact = polar(g, 5)
    off = (orthogonalize(g.cuda(), 5).cpu().double() - exact).norm()
    assert off <= polar_off(5) * exact.norm()


@pytest.mark.parametrize("tokens,dim", [(5, 33), (300, 33), (300, 1999)])
def test_captured_steps_of_odd_channels(tokens, dim):
    x, weight, targets, bias = _inputs(tokens, 1100, dim, BF16, bias=FP32, ignored=0.1)
    static = [t.cuda().requires_grad_() for t in (x, weight, bias)]
    at = targets.cuda()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = linear_cross_entropy(static[0], static[1], at, static[2], softcap=15.0)
        grads = torch.autograd.grad(out, static)
    for seed in (0, 3, 4):
        x, weight, targets, bias = _inputs(tokens, 1100, dim, BF16, bias=FP32, ignored=0.1,
                                           seed=seed)
        with torch.no_grad():
            for a, b in zip(static, (x, weight, bias)):
                a.copy_(b)
            at.copy_(targets)
        graph.replay()
        expected = _check(x, weight, targets, bias, softcap=15.0)
        torch.cuda.synchronize()
        assert torch.equal(out, expected[0]) and all(map(torch.equal, grads, expected[1]))


def test_calls_on_two_streams_at_once():
    cases = [[t.cuda() for t in _inputs(700, 3000, 128, BF16, bias=FP32, ignored=0.1, seed=s)]
             for s in range(2)]
    matrices = [_matrix((4, 300, 400), seed=s).to(BF16).cuda() for s in range(2)]

    def step(i):
        x, weight, targets, bias = cases[i]
        leaves = [t.detach().requires_grad_() for t in (x, weight, bias)]
        out = linear_cross_entropy(leaves[0], leaves[1], targets, leaves[2])
        return [out.detach(), *torch.autograd.grad(out, leaves), orthogonalize(matrices[i], 5)]

    alone = [step(i) for i in range(2)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(3):
        results = []
        for i, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                results.append(step(i))
        torch.cuda.synchronize()
        for a, b in zip(alone, results):
            assert all(map(torch.equal, a, b))


@pytest.mark.parametrize("tokens,dim", [(20, 64), (100, 33), (300, 64), (300, 2048)])
def test_memory_may_hold_anything(tokens, dim):
    """Results do not come from what working memory held: NaN everywhere first."""
    x, weight, targets, bias = _inputs(tokens, 513, dim, BF16, bias=FP32, ignored=0.2)
    g = _matrix((3, 133, 270)).to(BF16).cuda()
    plain, turned = _check(x, weight, targets, bias), orthogonalize(g, 5)
    for value in (float("nan"), float("inf")):
        torch.cuda.synchronize()
        torch.cuda.empty_cache()
        # What the next allocations are cut from.
        for size in (1 << 28, 1 << 20, 1 << 18, 1 << 10):
            memory = [torch.full((size,), value, dtype=BF16, device="cuda") for _ in range(4)]
            del memory
        again = _check(x, weight, targets, bias)
        assert torch.equal(plain[0], again[0]) and all(map(torch.equal, plain[1], again[1]))
        assert torch.equal(orthogonalize(g, 5), turned)
