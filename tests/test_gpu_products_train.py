"""The product operators in the trainer: the head's layer, Muon, and a step with both."""
from __future__ import annotations

import pytest
import torch

from examples.nanogpt import train_gpt_lct as trainer
from gpu_util import require_gpu
from losslessly_compressed_tensors_amd.LCTensor import LCTTensor
from losslessly_compressed_tensors_amd.components import layers
from losslessly_compressed_tensors_amd.components.losses import linear_cross_entropy
from losslessly_compressed_tensors_amd.components.orthogonal import orthogonalize
from losslessly_compressed_tensors_amd.components.sparse_utils import SparseMuon
from losslessly_compressed_tensors_amd.tensor_buffer import TensorBuffer
from product_oracle import polar, polar_off

pytestmark = pytest.mark.gpu
BF16, FP32 = torch.bfloat16, torch.float32


@pytest.fixture(autouse=True)
def _gpu():
    require_gpu()


def _head(tokens=256, vocab=1000, dim=512, seed=0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(2, tokens // 2, dim, generator=g).to(BF16)
    weight = (torch.randn(vocab, dim, generator=g) / dim ** 0.5).to(BF16)
    gain, bias = 1 + 0.1 * torch.randn(dim, generator=g), 0.1 * torch.randn(vocab, generator=g)
    targets = torch.randint(0, vocab, (2, tokens // 2), generator=g)
    targets[0, :5] = -100
    return [t.cuda() for t in (x, weight, gain, bias, targets)]


def _run_head(compressed=False, weight=None, reduction="sum"):
    x, w, gain, bias, targets = _head()
    leaves = [t.clone().requires_grad_() for t in (x, gain, bias)]
    if weight is None:
        weight = w.clone().requires_grad_()
    buffer = TensorBuffer(8 * 2 ** 20, device=x.device) if compressed else None
    out = layers.RMSLinearCrossEntropy.apply(
        leaves[0], weight, leaves[1], leaves[2], targets, buffer, compressed, layers.act_dist,
        1024, 15.0, -100, reduction)
    out.sum().backward()
    return out.detach(), [leaves[0].grad, weight.grad, leaves[1].grad, leaves[2].grad]


@pytest.mark.parametrize("reduction", ["sum", "mean", "none"])
def test_head_is_norm_then_loss(reduction):
    out, grads = _run_head(reduction=reduction)
    x, weight, gain, bias, targets = _head()
    y, rstd = layers._norm(x, gain)
    leaves = [t.requires_grad_() for t in (y, weight, bias)]
    expected = linear_cross_entropy(y, weight, targets, bias, softcap=15.0, reduction=reduction)
    grad_y, grad_weight, grad_bias = torch.autograd.grad(expected.sum(), leaves)
    grad_x, grad_gain, _ = layers._norm_backward(grad_y, x, rstd, gain)
    assert out.shape == expected.shape and torch.equal(out, expected.detach())
    for got, leaf in zip(grads, (grad_x, grad_weight, grad_gain, grad_bias)):
        assert got.dtype == leaf.dtype and torch.equal(got, leaf)


def test_head_with_its_input_compressed_is_the_same():
    plain, packed = _run_head(), _run_head(compressed=True)
    assert torch.equal(plain[0], packed[0])
    assert all(map(torch.equal, plain[1], packed[1]))


def test_head_with_a_compressed_weight_is_the_same():
    _, weight, *_ = _head()
    packed = LCTTensor(torch.nn.Parameter(weight), buffer=None, dist=layers.weight_dist)
    plain, got = _run_head(), _run_head(weight=packed)
    assert torch.equal(plain[0], got[0])
    assert all(map(torch.equal, plain[1], got[1]))


@pytest.mark.parametrize("frozen", [(0, 2), (1,), (3,), (1, 3)])
def test_head_with_frozen_inputs(frozen):
    _, grads = _run_head()
    x, weight, gain, bias, targets = _head()
    leaves = [t.requires_grad_(i not in frozen) for i, t in enumerate((x, weight, gain, bias))]
    layers.RMSLinearCrossEntropy.apply(*leaves[:4], targets, None, False, None, 1024,
                                       15.0).backward()
    for i, (leaf, grad) in enumerate(zip(leaves, grads)):
        assert leaf.grad is None if i in frozen else torch.equal(leaf.grad, grad)


def test_head_without_a_bias():
    x, weight, gain, _, targets = _head()
    leaves = [t.requires_grad_() for t in (x, weight, gain)]
    out = layers.RMSLinearCrossEntropy.apply(*leaves, None, targets)
    grads = torch.autograd.grad(out, leaves)
    y, _ = layers._norm(x.detach(), gain.detach())
    y.requires_grad_()
    expected = linear_cross_entropy(y, weight, targets, reduction="sum")
    assert torch.equal(out, expected)
    assert torch.equal(grads[1], torch.autograd.grad(expected, weight)[0])


def test_head_refuses_nothing_and_bad_targets():
    x, weight, gain, bias, targets = _head()
    with pytest.raises(ValueError, match="needs a token"):
        layers.RMSLinearCrossEntropy.apply(x[:0], weight, gain, bias, targets[:0])
    with pytest.raises(ValueError, match="targets must have shape"):
        layers.RMSLinearCrossEntropy.apply(x, weight, gain, bias, targets[:1])


def _muon(fused, compressed, shapes, seed=3):
    g = torch.Generator().manual_seed(seed)
    params = [torch.nn.Parameter(torch.randn(*s, generator=g).to(BF16).cuda()) for s in shapes]
    buffer = TensorBuffer(16 * 2 ** 20, device="cuda") if compressed else None
    muon = SparseMuon(params, lr=0.02, weight_decay=0.1, compressed=compressed, buffer=buffer,
                      ns_iters=5, fused=fused)
    for _ in range(3):
        for p in params:
            p.grad = torch.randn(p.shape, generator=g).to(BF16).cuda()
        muon.step()
    return [p.detach() for p in params]


SHAPES = [(256, 256), (256, 256), (512, 128), (128, 512), (512, 128), (4, 64, 72)]


def test_muon_with_compressed_momentum_is_the_same():
    for a, b in zip(_muon(True, False, SHAPES), _muon(True, True, SHAPES)):
        assert torch.equal(a, b)


def test_muons_direction_and_scale():
    """One step without momentum's history: p - lr times the scaled polar factor."""
    for shape in ((256, 128), (96, 160), (200, 200)):
        g = torch.randn(*shape, generator=torch.Generator().manual_seed(1)).to(BF16).cuda()
        p = torch.nn.Parameter(torch.zeros(*shape, dtype=BF16, device="cuda"))
        p.grad = g.clone()
        SparseMuon([p], lr=1.0, mu=0.0, compressed=False, ns_iters=8, fused=True).step()
        scale = max(1.0, shape[0] / shape[1]) ** 0.5
        exact = -polar(g.cpu(), 8, scale)
        off = (p.detach().cpu().double() - exact).norm()
        assert off <= polar_off(8) * exact.norm()
        assert torch.equal(p.detach(), -orthogonalize(g, 8, scale=scale))


def test_muon_near_the_librarys_iteration():
    """The library's is in BF16: 13 roundings of 2^-9 a step, independent ones."""
    for a, b in zip(_muon(True, False, SHAPES), _muon(False, False, SHAPES)):
        start = a.float().norm()
        assert (a.float() - b.float()).norm() <= 0.02 * 3 * 0.1 * start


def _model(**options):
    return trainer.build(torch.device("cuda:0"), vocab_size=512, num_layers=2, model_dim=128,
                         head_dim=64, buffer_mib=16, **options)


def _step(options, compressed, steps=2):
    model, optimizers = _model(compress_weights=False, compress_activations=compressed,
                               compress_optimizer=compressed, **options)
    losses = []
    for i in range(steps):
        inputs, targets = trainer.random_tokens(4, 256, "cuda", seed=i, token_ids=512)
        losses.append(trainer.train_step(model, optimizers, inputs, targets))
    return losses, {n: p.detach().clone() for n, p in model.named_trainable_tensors()}


def test_a_step_with_both_compressed_is_the_same():
    options = dict(fused_head=True, fused_muon=True)
    plain, packed = _step(options, False), _step(options, True)
    assert all(map(torch.equal, plain[0], packed[0]))
    for name, p in plain[1].items():
        assert torch.equal(p, packed[1][name]), name


def test_a_step_with_compressed_weights_runs():
    model, optimizers = _model(compress_weights=True, compress_activations=True,
                               compress_optimizer=True, fused_head=True, fused_muon=True,
                               window=64, sinks=2, dropout=0.1)
    inputs, targets = trainer.random_tokens(4, 256, "cuda", seed=0, token_ids=512)
    for _ in range(2):
        assert trainer.train_step(model, optimizers, inputs, targets).isfinite()


def test_the_heads_gradients_against_the_default_head():
    """The default head rounds logits below 2^4 to BF16, 2^-5 apart: a probability moves by
    that much at most, and so does its row's gradient."""
    grads = {}
    for fused in (False, True):
        torch.manual_seed(0)
        model, _ = _model(compress_weights=False, compress_activations=False,
                          compress_optimizer=False, fused_head=fused)
        with torch.no_grad():
            for name, p in model.named_parameters():
                if "proj" in name and name.endswith("weight"):
                    p.normal_(std=p.shape[-1] ** -0.5,
                              generator=torch.Generator("cuda").manual_seed(1))
        inputs, targets = trainer.random_tokens(2, 128, "cuda", seed=5, token_ids=512)
        loss = model(inputs, targets)
        loss.backward()
        grads[fused] = float(loss.detach()), {n: p.grad.float() for n, p
                                              in model.named_trainable_tensors()}
    assert abs(grads[True][0] - grads[False][0]) <= 2.0 ** -6 * grads[False][0]
    for name, g in grads[False][1].items():
        assert (g - grads[True][1][name]).norm() <= 2.0 ** -5 * g.norm(), name


def test_options_leave_the_default_step_as_it_was():
    default, spelled = _step({}, False), _step(dict(fused_head=False, fused_muon=False), False)
    assert all(map(torch.equal, default[0], spelled[0]))


def test_no_logits_are_kept():
    """The head's step allocates less than its logits alone would take."""
    tokens, vocab, dim = 4096, 50304, 256
    x = torch.randn(tokens, dim, device="cuda").to(BF16).requires_grad_()
    weight = torch.randn(vocab, dim, device="cuda").mul_(0.1).to(BF16).requires_grad_()
    targets = torch.randint(0, vocab, (tokens,), device="cuda")
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    linear_cross_entropy(x, weight, targets).backward()
    peak = torch.cuda.max_memory_allocated() - before
    # In 16 bits: 393 MiB.  Here: a piece of their gradient, parts, sums, both gradients.
    assert peak < 2 * tokens * vocab


@pytest.mark.parametrize("reduction", ["sum", "none"])
def test_heads_gradients_are_no_constants(reduction):
    """A second derivative is refused: neither the loss's kernels nor the norm's saved values
    have one."""
    values = _head()
    for at in range(4):
        leaves = [t.detach().clone().requires_grad_(i == at) for i, t in enumerate(values[:4])]

        def loss():
            return layers.RMSLinearCrossEntropy.apply(*leaves, values[4], None, False, None, 1024,
                                                      15.0, -100, reduction).sum()

        plain, = torch.autograd.grad(loss(), leaves[at])
        out = loss()
        grad, = torch.autograd.grad(out, leaves[at], create_graph=True)
        assert torch.equal(grad, plain)
        with pytest.raises(RuntimeError, match="differentiated once only"):
            grad.float().square().sum().backward()


def test_changed_inputs_of_the_head_are_noticed():
    x, weight, gain, bias, targets = _head()
    leaf, hidden = gain.requires_grad_(), x.clone()
    out = layers.RMSLinearCrossEntropy.apply(hidden, weight, leaf, bias, targets)
    hidden.zero_()
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        out.backward()


def test_a_second_backward_pass_of_the_head():
    """An input that is not compressed is still there; a compressed one was freed."""
    for compressed in (False, True):
        x, weight, gain, bias, targets = _head()
        leaves = [t.requires_grad_() for t in (x, weight, gain, bias)]
        buffer = TensorBuffer(8 * 2 ** 20, device=x.device) if compressed else None
        out = layers.RMSLinearCrossEntropy.apply(*leaves, targets, buffer, compressed,
                                                 layers.act_dist, 1024)
        first = torch.autograd.grad(out, leaves, retain_graph=True)
        if compressed:
            with pytest.raises(RuntimeError, match="freed by an earlier backward pass"):
                out.backward()
        else:
            assert all(map(torch.equal, first, torch.autograd.grad(out, leaves)))


@pytest.mark.parametrize("compressed", [False, True])
def test_a_refused_step_of_muon_changes_nothing(compressed):
    shapes = [(256, 128), ((1 << 16) + 1, 2)]
    g = torch.Generator().manual_seed(0)
    params = [torch.nn.Parameter(torch.randn(*s, generator=g).to(BF16).cuda()) for s in shapes]
    buffer = TensorBuffer(16 * 2 ** 20, device="cuda") if compressed else None
    muon = SparseMuon(params, compressed=compressed, buffer=buffer, fused=True)
    params[0].grad = torch.randn(*shapes[0], generator=g).to(BF16).cuda()
    muon.step()
    for p in params:
        p.grad = torch.randn(p.shape, generator=g).to(BF16).cuda()

    def held():
        momenta = [m.decompress() if isinstance(m, LCTTensor) else m
                   for m in muon.momentums if m is not None]
        return [t.detach().clone() for t in (*params, *(p.grad for p in params), *momenta)]

    before = held()
    with pytest.raises(ValueError, match="at most 65536 rows"):
        muon.step()
    assert len(before) == len(held()) and all(map(torch.equal, before, held()))
    muon.ns_iters = 1001
    params[1].grad = None
    with pytest.raises(ValueError, match="steps"):
        muon.step()
    muon.ns_iters = 5
    muon.step()
    assert not torch.equal(before[0], params[0])


@pytest.mark.parametrize("compressed", [False, True])
@pytest.mark.parametrize("value", [float("nan"), float("inf"), -3e38])
def test_what_ignored_tokens_hold_reaches_nothing_of_the_head(value, compressed):
    results = []
    for dirty in (False, True):
        x, weight, gain, bias, targets = _head()
        if dirty:
            x[targets == -100] = value
        held = x.clone()
        leaves = [t.requires_grad_() for t in (x, weight, gain, bias)]
        buffer = TensorBuffer(8 * 2 ** 20, device=x.device) if compressed else None
        out = layers.RMSLinearCrossEntropy.apply(*leaves, targets, buffer, compressed,
                                                 layers.act_dist, 1024, 15.0)
        results.append([out.detach(), *torch.autograd.grad(out, leaves)])
        assert torch.equal(x.detach().view(torch.int16), held.view(torch.int16))
    assert (targets == -100).any() and not results[1][1][targets == -100].any()
    assert all(map(torch.equal, *results))
