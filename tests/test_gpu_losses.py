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


# From 2048 channels and 129 tokens on, the logits' tiles are 256 x 256.
@pytest.mark.parametrize("softcap", [None, 15.0])
@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("tokens,vocab,dim", [(128, 300, 2048), (129, 255, 2048), (257, 513, 2056),
                                              (300, 1100, 4096)])
def test_deep_products(tokens, vocab, dim, dtype, softcap):
    x, weight, targets, bias = _inputs(tokens, vocab, dim, dtype, bias=FP32)
    _check(x, weight, targets, bias if softcap else None, softcap=softcap)


@pytest.mark.parametrize("dim", [1, 2, 7, 13, 33, 70, 129])
def test_odd_channels(dim):
    x, weight, targets, bias = _inputs(21, 67, dim, BF16, bias=FP32)
    _check(x, weight, targets, bias, reduction="sum")


def test_odd_channels_of_many_words():
    # (Matrices of a million values are widened another way.)
    x, weight, targets, bias = _inputs(130, 8200, 129, BF16, bias=FP32)
    _check(x, weight, targets, bias)


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


def test_layouts():
    """Leading dimensions, strided and misaligned rows, strided targets and bias."""
    x, weight, targets, bias = _inputs(2 * 3 * 17, 131, 64, BF16, bias=FP32)
    base, grads = _check(x, weight, targets, bias)
    x3 = x.view(2, 3, 17, 64)
    out, _ = _check(x3, weight, targets.view(2, 3, 17), bias)
    assert torch.equal(out, base)
    wide = torch.randn(x.shape[0], 192).to(BF16).cuda()
    wide[:, 64:128] = x
    tall = torch.randn(64, 131).to(BF16).cuda()
    tall.copy_(weight.T)
    odd = torch.randn(x.shape[0] * 64 + 1).to(BF16).cuda()
    odd[1:] = x.reshape(-1)
    for xs in (wide[:, 64:128], odd[1:].view(-1, 64), x.cuda()):
        for ws in (tall.T, weight.cuda()):
            for ts in (targets.cuda(), targets.repeat_interleave(2).cuda()[::2]):
                for bs in (bias.cuda(), bias.repeat_interleave(3).cuda()[::3]):
                    assert torch.equal(linear_cross_entropy(xs, ws, ts, bs), base)


def test_bias_of_the_inputs_type():
    for dtype in (BF16, FP16):
        x, weight, targets, bias = _inputs(50, 300, 32, dtype, bias=dtype)
        _, grads = _check(x, weight, targets, bias)
        full = CrossEntropy(x, weight, targets, bias)
        u = torch.finfo(dtype).eps / 2
        assert_within(grads[2], full.grad_bias,
                      full.grad_bias_off + u * full.grad_bias.abs() + torch.finfo(dtype).tiny, "bias")


@pytest.mark.parametrize("frozen", [(0,), (1,), (2,), (0, 1), (0, 2), (1, 2)])
def test_gradients_that_are_not_needed(frozen):
    x, weight, targets, bias = _inputs(300, 513, 64, BF16, bias=FP32)
    _, all_grads = _check(x, weight, targets, bias)
    leaves = [t.cuda().requires_grad_(i not in frozen) for i, t in enumerate((x, weight, bias))]
    linear_cross_entropy(leaves[0], leaves[1], targets.cuda(), leaves[2]).backward()
    for i, leaf in enumerate(leaves):
        assert leaf.grad is None if i in frozen else torch.equal(leaf.grad, all_grads[i])


@pytest.mark.parametrize("softcap", [None, 30.0])
def test_results_do_not_depend_on_the_run(softcap):
    x, weight, targets, bias = _inputs(700, 1501, 136, BF16, bias=FP32, ignored=0.2)
    first = _check(x, weight, targets, bias, softcap=softcap)
    for _ in range(3):
        again = _check(x, weight, targets, bias, softcap=softcap)
        assert torch.equal(first[0], again[0])
        assert all(torch.equal(a, b) for a, b in zip(first[1], again[1]))


def test_what_ignored_tokens_hold_reaches_nothing():
    x, weight, targets, bias = _inputs(300, 257, 64, BF16, bias=FP32, ignored=0.3)
    plain = _check(x, weight, targets, bias)
    dirty = x.clone()
    ignored = targets == -100
    dirty[ignored] = torch.tensor([float("nan"), float("inf"), -float("inf"), 3e38]).to(
        BF16).repeat(16)
    out = _check(dirty, weight, targets, bias)
    assert torch.equal(plain[0], out[0])
    assert all(torch.equal(a, b) for a, b in zip(plain[1], out[1]))
    assert not out[1][0][ignored.cuda()].any()
    for few in (3, 30, 200):
        rows = ignored.nonzero()[:1].flatten().tolist() + list(range(few - 1))
        none = linear_cross_entropy(dirty[rows].cuda(), weight.cuda(), targets[rows].cuda(),
                                    bias.cuda(), reduction="none")
        assert none.isfinite().all() and none[0] == 0


def test_another_ignored_index_may_be_a_word():
    x, weight, targets, bias = _inputs(90, 40, 32, BF16, bias=FP32)
    assert (targets == 7).any()
    _check(x, weight, targets, bias, ignore_index=7)
    _check(x, weight, targets, bias, ignore_index=2 ** 40)


def test_targets_outside_the_vocabulary_give_nan():
    x, weight, targets, bias = _inputs(40, 90, 32, BF16, bias=FP32)
    for bad in (-1, 90, 2 ** 31 + 5, -2 ** 40):
        wrong = targets.clone()
        wrong[3] = bad
        losses = linear_cross_entropy(x.cuda(), weight.cuda(), wrong.cuda(), bias.cuda(),
                                      reduction="none")
        assert losses[3].isnan() and losses[torch.arange(40) != 3].isfinite().all()
        _check(x, weight, wrong, bias)


def test_no_tokens():
    weight = torch.randn(9, 16).to(BF16).cuda().requires_grad_()
    for shape in ((0,), (3, 0)):
        x = torch.zeros(*shape, 16, dtype=BF16, device="cuda", requires_grad=True)
        targets = torch.zeros(shape, dtype=torch.int64, device="cuda")
        for reduction in ("mean", "sum", "none"):
            out = linear_cross_entropy(x, weight, targets, reduction=reduction)
            assert out.shape == (shape if reduction == "none" else ()) and not out.any()
            weight.grad = None
            out.sum().backward()
            assert not weight.grad.any() and x.grad.shape == x.shape


@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_biases_that_take_words_out(dtype):
    """-inf and the lowest FP32 number: probability zero, gradients zero; rows that are left
    with their target alone."""
    x, weight, targets, bias = _inputs(70, 300, 32, dtype, bias=FP32)
    for low in (-float("inf"), torch.finfo(FP32).min):
        masked = bias.clone()
        masked[130:] = low
        inside = targets % 130
        _, grads = _check(x, weight, inside, masked)
        assert not grads[1][130:].any()
        alone = torch.full_like(bias, low)
        alone[11] = 0.5
        out = linear_cross_entropy(x.cuda(), weight.cuda(), torch.full((70,), 11).cuda(),
                                   alone.cuda(), reduction="none")
        assert not out.any()


def test_a_target_that_is_taken_out():
    x, weight, targets, bias = _inputs(20, 50, 32, BF16, bias=FP32)
    bias[4] = -float("inf")
    targets[:] = 3
    targets[2] = 4
    out = linear_cross_entropy(x.cuda(), weight.cuda(), targets.cuda(), bias.cuda(),
                               reduction="none")
    assert out[2] == float("inf") and out[torch.arange(20) != 2].isfinite().all()
    leaves = [t.cuda().requires_grad_() for t in (x, weight)]
    linear_cross_entropy(*leaves, targets.cuda(), bias.cuda(), reduction="sum").backward()
    exact = CrossEntropy(x, weight, torch.where(targets == 4, -100, targets), bias,
                         reduction="sum")
    # The others' gradients, and of the one a softmax less one.
    row = torch.arange(20) != 2
    assert_within(leaves[0].grad[row.cuda()], exact.grad_x[row], exact.grad_x_off[row], "grad_x")
    assert leaves[0].grad.isfinite().all() and leaves[1].grad.isfinite().all()


def test_infinite_and_nan_logits():
    x, weight, targets, bias = _inputs(40, 90, 32, BF16, bias=FP32)
    x[5, 3] = float("nan")
    x[7] = float("inf")
    losses = linear_cross_entropy(x.cuda(), weight.cuda(), targets.cuda(), bias.cuda(),
                                  reduction="none")
    bad = torch.zeros(40, dtype=torch.bool)
    bad[[5, 7]] = True
    assert torch.equal(losses.isnan().cpu(), bad)


def test_logits_far_past_the_cap():
    """z^2 does not fit FP32: capped at s, with no gradient."""
    x, weight, targets, bias = _inputs(40, 90, 32, BF16, bias=FP32)
    for far in (1e30, -1e30, float("inf"), torch.finfo(FP32).min):
        bias[8] = far
        capped = bias.clone()
        # s (1 - 1e-9) is s in FP32: 15 for the oracle too.
        capped[8] = 1e9 if far > 0 else -1e9
        exact = CrossEntropy(x, weight, targets, capped, 15.0, reduction="none")
        exact.losses_off += 1e-6
        out = linear_cross_entropy(x.cuda(), weight.cuda(), targets.cuda(), bias.cuda(),
                                   softcap=15.0, reduction="none")
        assert_within(out, exact.losses, exact.losses_off, "losses")
        leaves = [t.cuda().requires_grad_() for t in (x, weight, bias)]
        linear_cross_entropy(leaves[0], leaves[1], targets.cuda(), leaves[2], softcap=15.0,
                             reduction="sum").backward()
        assert all(leaf.grad.isfinite().all() for leaf in leaves)
        assert not leaves[1].grad[8].any() and leaves[2].grad[8] == 0


@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_sure_and_unsure_targets(dtype):
    """Losses from 1e-30 to 80: relative precision where the target is sure."""
    g = torch.Generator().manual_seed(5)
    weight = torch.randn(200, 64, generator=g).to(dtype)
    targets = torch.randint(0, 200, (120,), generator=g)
    size = torch.linspace(-1, 1, 120)[:, None]
    x = (size * weight[targets].float()).to(dtype)
    out, _ = _check(x, weight, targets, reduction="none", grad=torch.ones(120))
    assert out.min() < 1e-10 and out.max() > 60


def test_gradients_against_differences():
    x, weight, targets, bias = _inputs(9, 21, 16, BF16, bias=FP32, spread=1.0)
    leaf = bias.cuda().requires_grad_()
    linear_cross_entropy(x.cuda(), weight.cuda(), targets.cuda(), leaf, softcap=5.0,
                         reduction="sum").backward()
    h = 2.0 ** -4
    for v in range(21):
        ends = []
        for sign in (1, -1):
            moved = bias.clone()
            moved[v] += sign * h
            ends.append(float(linear_cross_entropy(x.cuda(), weight.cuda(), targets.cuda(),
                                                   moved.cuda(), softcap=5.0, reduction="sum")))
        # A third derivative below 2 per token, and FP32's rounding of losses below 64.
        assert abs((ends[0] - ends[1]) / (2 * h) - float(leaf.grad[v])) \
            < 9 * 2 * h * h / 6 + 2 * 64 * 2.0 ** -24 / h


def test_losses_none_belong_to_the_caller():
    x, weight, targets, bias = _inputs(30, 60, 32, BF16, bias=FP32)
    leaves = [t.cuda().requires_grad_() for t in (x, weight)]
    out = linear_cross_entropy(*leaves, targets.cuda(), reduction="none")
    grads = torch.autograd.grad(out.sum(), leaves, retain_graph=True)
    with torch.no_grad():
        out.zero_()
    again = torch.autograd.grad(out.sum(), leaves)
    assert all(torch.equal(a, b) for a, b in zip(grads, again))


def test_changed_inputs_are_noticed():
    x, weight, targets, _ = _inputs(30, 60, 32, BF16)
    leaf, w = x.cuda().requires_grad_(), weight.cuda()
    out = linear_cross_entropy(leaf, w, targets.cuda())
    w.zero_()
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        out.backward()


def test_second_derivatives_are_refused():
    x, weight, targets, _ = _inputs(30, 60, 32, BF16)
    leaf = x.cuda().requires_grad_()
    out = linear_cross_entropy(leaf, weight.cuda(), targets.cuda())
    grad, = torch.autograd.grad(out, leaf, create_graph=True)
    with pytest.raises(RuntimeError):
        grad.sum().backward()


def test_streams_and_replays():
    """On another stream, and captured: replays with new contents, eager work between."""
    x, weight, targets, bias = _inputs(300, 1000, 64, BF16, bias=FP32, ignored=0.2)
    eager = _check(x, weight, targets, bias, softcap=15.0)
    side = torch.cuda.Stream()
    leaves = [t.cuda().requires_grad_() for t in (x, weight, bias)]
    at = targets.cuda()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        out = linear_cross_entropy(leaves[0], leaves[1], at, leaves[2], softcap=15.0)
        grads = torch.autograd.grad(out, leaves)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    assert torch.equal(out, eager[0]) and all(map(torch.equal, grads, eager[1]))

    static = [t.detach().clone().requires_grad_() for t in leaves]
    static_targets = at.clone()
    graphs = []
    for _ in range(2):      # two graphs: each has its own workspaces
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = linear_cross_entropy(static[0], static[1], static_targets, static[2],
                                       softcap=15.0)
            grads = torch.autograd.grad(out, static)
        graphs.append((graph, out, grads))
    for seed in (0, 3, 4):
        x, weight, targets, bias = _inputs(300, 1000, 64, BF16, bias=FP32,
                                           ignored=0.1 * seed, seed=seed)
        with torch.no_grad():
            for a, b in zip(static, (x, weight, bias)):
                a.copy_(b)
            static_targets.copy_(targets)
        for graph, _, _ in graphs:
            graph.replay()
        expected = _check(x, weight, targets, bias, softcap=15.0)
        torch.cuda.synchronize()
        for graph, out, grads in graphs:
            assert torch.equal(out, expected[0]) and all(map(torch.equal, grads, expected[1]))


def test_refusals():
    x, weight, targets, bias = (t.cuda() for t in _inputs(6, 10, 16, BF16, bias=FP32))
    calls = [
        (dict(x=x.float()), TypeError), (dict(weight=weight.half()), TypeError),
        (dict(weight=weight[0]), ValueError), (dict(weight=weight[:, :8]), ValueError),
        (dict(weight=weight[:0]), ValueError), (dict(weight=weight.cpu()), ValueError),
        (dict(targets=targets.float()), TypeError), (dict(targets=targets[:3]), ValueError),
        (dict(targets=targets.cpu()), ValueError), (dict(bias=bias[:4]), ValueError),
        (dict(bias=bias.double()), TypeError), (dict(bias=bias.cpu()), ValueError),
        (dict(softcap=0.0), ValueError), (dict(softcap=-1.0), ValueError),
        (dict(softcap=float("inf")), ValueError), (dict(reduction="all"), ValueError),
        (dict(ignore_index=0.5), TypeError), (dict(ignore_index=2 ** 63), ValueError),
        (dict(x=x[:, :0], weight=weight[:, :0]), ValueError),
    ]
    for changes, error in calls:
        args = dict(x=x, weight=weight, targets=targets, bias=bias)
        args.update(changes)
        with pytest.raises(error):
            linear_cross_entropy(**args)
    # Nothing is allocated for them.
    few = torch.zeros(1, 8, dtype=BF16, device="cuda")
    with pytest.raises(ValueError, match="tokens times vocabulary"):
        linear_cross_entropy(few.expand(1 << 22, 8), few.expand((1 << 15) + 1, 8),
                             targets.new_zeros(1).expand(1 << 22))
    with pytest.raises(RuntimeError, match="recorded"):
        torch.jit.trace(lambda a: linear_cross_entropy(a, weight, targets), x)
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(x, torch.ones_like(x))
        with pytest.raises(RuntimeError, match="forward-mode"):
            linear_cross_entropy(dual, weight, targets)


@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_several_pieces_and_many_token_tiles(dtype, monkeypatch):
    """Pieces and splits as large calls have them, at a size the oracle can check."""
    from losslessly_compressed_tensors_amd.kernels import products
    x, weight, targets, bias = _inputs(600, 2000, 96, dtype, bias=FP32, ignored=0.1)
    for piece, splits in ((256, 1), (512, 3), (768, 16), (2048, 7)):
        monkeypatch.setattr(products, "vocabulary_pieces", lambda *a: (piece, splits))
        _check(x, weight, targets, bias, softcap=30.0)


@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_several_pieces_of_few_tokens(dtype, monkeypatch):
    from losslessly_compressed_tensors_amd.kernels import products
    x, weight, targets, bias = _inputs(101, 2000, 96, dtype, bias=FP32, ignored=0.1)
    for piece, splits in ((256, 1), (512, 3), (768, 32), (2048, 7)):
        monkeypatch.setattr(products, "vocabulary_pieces", lambda *a: (piece, splits))
        _check(x, weight, targets, bias, softcap=30.0)


@pytest.mark.parametrize("tokens", [1, 100, 200])
def test_many_parts(tokens):
    x, weight, targets, bias = _inputs(tokens, 17000, 64, BF16, bias=FP32)
    _check(x, weight, targets, bias, reduction="sum")


# Up to 128 tokens, and more: other tiles of all products.
@pytest.mark.parametrize("tokens", [40, 150])
def test_offsets_past_32_bits(tokens):
    """A vocabulary's matrix, and its gradient, of more than 2^32 bytes."""
    dim, vocab = 4096, (1 << 19) + 321
    weight = torch.zeros(vocab, dim, dtype=BF16, device="cuda")
    x = torch.zeros(tokens, dim, dtype=BF16, device="cuda")
    x[:, 0] = 1.0
    weight[:, 0] = torch.linspace(-4, 4, vocab, device="cuda").to(BF16)
    targets = torch.arange(vocab - tokens, vocab, device="cuda")
    leaves = [x.requires_grad_(), weight.requires_grad_()]
    out = linear_cross_entropy(*leaves, targets, reduction="sum")
    grads = torch.autograd.grad(out, leaves)
    z = weight.detach()[:, 0].double()
    lse = torch.logsumexp(z, 0)
    exact = tokens * lse - z[targets].sum()
    assert abs(float(out) - float(exact)) < 1e-4 * float(exact)
    p = tokens * (z - lse).exp()
    p[targets] -= 1.0
    assert_within(grads[1][:, 0], p.cpu(), (2.0 ** -6 * p.abs() + 1e-12).cpu(), "grad_weight")
    assert not grads[1][:, 1:].any()


@pytest.mark.parametrize("reduction", ["mean", "none"])
def test_gradients_of_a_loss_are_no_constants(reduction):
    """The incoming gradient is one here, which needs no gradient: a penalty on the loss's
    gradient is refused, not left out."""
    x, weight, targets, bias = _inputs(30, 60, 32, BF16, bias=FP32)
    for at in range(3):
        leaves = [t.cuda().requires_grad_(i == at) for i, t in enumerate((x, weight, bias))]
        loss = linear_cross_entropy(leaves[0], leaves[1], targets.cuda(), leaves[2],
                                    reduction=reduction)
        plain, = torch.autograd.grad(loss.sum(), leaves[at], retain_graph=True)
        grad, = torch.autograd.grad(loss.sum(), leaves[at], create_graph=True)
        assert torch.equal(grad, plain)
        with pytest.raises(RuntimeError, match="differentiated once only"):
            (loss.sum() + grad.float().square().sum()).backward()
