"""Rotary positions and the caches' writes against complex multiplication in 64
bits (``attention_oracle``)."""
from __future__ import annotations

from fractions import Fraction

import attention_oracle as oracle
import pytest
import torch

from losslessly_compressed_tensors_amd.components import attention

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32


def _values(*shape, dtype=BF16, seed=0):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(dtype).to(DEV)


def _near(got, x, positions, frequencies, dtype, **how):
    exact = oracle.turned(x, positions, frequencies, **how)
    how.pop("back", None)
    bound = oracle.turned_bound(x, dtype, exact, frequencies, **how)
    assert got.dtype == dtype and got.shape == exact.shape
    far = (got.detach().cpu().double() - exact).abs() - bound
    assert bool((far <= 0).all()), float(far.max())


def _positions(batch, tokens, start):
    return torch.arange(tokens).expand(batch, tokens) + torch.as_tensor(start).reshape(-1, 1)


# batch, tokens, heads, key heads, channels, turned channels
SHAPES = [(1, 1, 1, 1, 8, 8), (2, 17, 12, 12, 64, 64), (3, 5, 4, 2, 128, 64), (1, 33, 3, 1, 80, 40),
          (2, 3, 2, 2, 10, 6), (1, 2, 5, 1, 7, 2), (1, 700, 2, 1, 96, 96), (2, 9, 1, 1, 256, 256)]


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "x".join(map(str, s)))
def test_rotation_and_gradient(shape, interleaved, dtype):
    batch, tokens, heads, kv_heads, dim, turned = shape
    frequencies = attention.rotary_frequencies(turned)
    plan = attention.Rotary(frequencies, interleaved=interleaved, magnitude=1.25)
    q = _values(batch, tokens, heads, dim, dtype=dtype).requires_grad_()
    k = _values(batch, tokens, kv_heads, dim, dtype=dtype, seed=1).requires_grad_()
    grads = _values(batch, tokens, heads, dim, dtype=dtype, seed=2), _values(
        batch, tokens, kv_heads, dim, dtype=dtype, seed=3)
    out = attention.apply_rotary(plan, q, k, positions=41)
    back = torch.autograd.grad(out, (q, k), grads)
    how = {"interleaved": interleaved, "magnitude": 1.25}
    at = _positions(batch, tokens, 41)
    for x, got, grad, grad_in in zip((q, k), out, grads, back):
        _near(got, x, at, frequencies, dtype, **how)
        _near(grad_in, grad, at, frequencies, dtype, back=True, **how)
        assert torch.equal(got[..., turned:], x[..., turned:])
    # A rotation is linear: differences of any step are its own values.
    step = oracle.turned(q, at, frequencies, **how) - oracle.turned(0.5 * q, at, frequencies, **how)
    dot = (grads[0].cpu().double() * 2 * step).sum()
    size = (back[0].cpu().double() * q.detach().cpu().double()).abs().sum()
    assert abs((back[0].cpu().double() * q.detach().cpu().double()).sum() - dot) \
        <= (oracle.UNIT[dtype] + 64 * oracle.STEP) * size + 1e-6
    alone = attention.apply_rotary(plan, q.detach(), positions=41)
    assert torch.equal(alone, out[0])


@pytest.mark.parametrize("kind", ["none", "integer", "starts", "each", "far", "negative", "int64"])
def test_positions(kind):
    q, k = _values(3, 21, 4, 64, dtype=FP32), _values(3, 21, 2, 64, dtype=FP32, seed=1)
    frequencies = attention.rotary_frequencies(64, scaling="ramp", factor=8.0)
    plan = attention.Rotary(frequencies)
    starts = torch.tensor([5, 70000, 2])
    each = torch.randint(0, 1 << 17, (3, 21), generator=torch.Generator().manual_seed(1))
    given, at = {
        "none": (None, _positions(3, 21, 0)), "integer": (9000, _positions(3, 21, 9000)),
        "starts": (starts.int().to(DEV), _positions(3, 21, starts)),
        "each": (each.int().to(DEV), each),
        "far": (1 << 30, _positions(3, 21, 1 << 30)), "negative": (-77, _positions(3, 21, -77)),
        "int64": (each.to(DEV), each)}[kind]
    got = attention.apply_rotary(plan, q, k, positions=given)
    # FP64 angles at 2^30 are themselves good to 2^-23 of a radian.
    for x, y in zip((q, k), got):
        exact = oracle.turned(x, at, frequencies)
        bound = oracle.turned_bound(x, FP32, exact, frequencies)
        if kind == "far":
            bound = bound + 2.0 ** -22 * 2 * x.cpu().double().abs().amax()
        assert bool(((y.cpu().double() - exact).abs() <= bound).all())


def test_broadcast_positions():
    """One position for all tokens of a sequence, or one row for all sequences."""
    q = _values(3, 6, 2, 64, dtype=FP32)
    plan = attention.Rotary(attention.rotary_frequencies(64))
    for given in (torch.tensor([[7], [1], [0]], dtype=torch.int32, device=DEV).expand(3, 6),
                  torch.arange(6, dtype=torch.int32, device=DEV).expand(3, 6),
                  torch.tensor([9], dtype=torch.int32, device=DEV).expand(3)):
        assert torch.equal(attention.apply_rotary(plan, q, positions=given),
                           attention.apply_rotary(plan, q, positions=given.contiguous()))
    same = torch.tensor([[7], [1], [0]], dtype=torch.int32, device=DEV).expand(3, 6)
    _near(attention.apply_rotary(plan, q, positions=same), q, same,
          attention.rotary_frequencies(64), FP32)


def test_the_trainers_rotation():
    """The frequencies of the trainer's eager form, and its sense."""
    from examples.nanogpt.train_gpt_lct import Rotary
    x = _values(2, 300, 3, 64, dtype=FP32)
    plan = attention.Rotary(attention.trainer_frequencies(64))
    eager = Rotary(64).to(DEV)(x)
    got = attention.apply_rotary(plan, x)
    # The eager form's FP32 angles: 300 positions times 2^-24, and its powers' 2^-22.
    assert bool(((got - eager).abs() <= 300 * 2.0 ** -21 * x.abs().amax()).all())


def test_strides_and_one_sided_gradients():
    both = _values(2, 40, 6, 64)
    q, k = both[:, :, :4].requires_grad_(), both[:, :, 4:].detach().requires_grad_()
    plan = attention.Rotary(attention.rotary_frequencies(64))
    want = attention.apply_rotary(plan, q.detach().contiguous(), k.detach().contiguous())
    rq, rk = attention.apply_rotary(plan, q, k)
    assert torch.equal(rq, want[0]) and torch.equal(rk, want[1])
    gk, = torch.autograd.grad(rk.float().sum(), k, retain_graph=True)
    gq, = torch.autograd.grad(rq.float().sum(), q)
    assert gk.shape == k.shape and gq.shape == q.shape
    head_major = _values(2, 4, 40, 64, seed=3).transpose(1, 2)
    assert torch.equal(attention.apply_rotary(plan, head_major),
                       attention.apply_rotary(plan, head_major.contiguous()))
    broken = _values(2, 40, 64, 4, seed=4).transpose(2, 3)
    assert torch.equal(attention.apply_rotary(plan, broken),
                       attention.apply_rotary(plan, broken.contiguous()))
    odd = torch.zeros(2 * 40 * 4 * 64 + 1, dtype=BF16, device=DEV)[1:].view(2, 40, 4, 64)
    odd.copy_(head_major)
    assert torch.equal(attention.apply_rotary(plan, odd), attention.apply_rotary(plan, head_major))
    empty = _values(2, 0, 4, 64)
    assert attention.apply_rotary(plan, empty, empty[:, :, :2])[1].shape == (2, 0, 2, 64)


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("batch,heads,kv_heads,dim,turned,interleaved",
                         [(1, 12, 12, 64, 64, False), (5, 8, 2, 128, 64, True),
                          (3, 2, 1, 10, 6, False)])
def test_append(batch, heads, kv_heads, dim, turned, interleaved, dtype):
    capacity = 37
    frequencies = attention.rotary_frequencies(turned)
    plan = attention.Rotary(frequencies, interleaved=interleaved)
    q = _values(batch, heads, dim, dtype=dtype)
    k, v = (_values(batch, kv_heads, dim, dtype=dtype, seed=s) for s in (1, 2))
    caches = [_values(batch, capacity, kv_heads, dim, dtype=dtype, seed=s) for s in (3, 4)]
    before = [c.clone() for c in caches]
    at = torch.tensor([36, 0, 17, -1, 37][:batch])
    got = attention.rotary_append(plan, q, k, v, *caches, at.int().to(DEV))
    _near(got.unsqueeze(1), q.unsqueeze(1), at.unsqueeze(1), frequencies, dtype,
          interleaved=interleaved)
    turned_k = attention.apply_rotary(plan, k.unsqueeze(1), positions=at.to(DEV)).squeeze(1)
    for b, p in enumerate(at.tolist()):
        if 0 <= p < capacity:
            before[0][b, p], before[1][b, p] = turned_k[b], v[b]
    assert torch.equal(caches[0], before[0]) and torch.equal(caches[1], before[1])


def test_frequencies():
    plain = attention.rotary_frequencies(64)
    assert float(plain[0]) == 1 and abs(float(plain[16]) - 0.01) < 1e-15
    assert torch.equal(attention.rotary_frequencies(64, scaling="linear", factor=4), plain / 4)
    raised = attention.rotary_frequencies(64, scaling="base", factor=4)
    assert float(raised[0]) == 1 and abs(float(raised[-1] / plain[-1]) - 0.25) < 1e-12
    ramp = attention.rotary_frequencies(64, scaling="ramp", factor=4)
    assert float(ramp[0]) == 1 and abs(float(ramp[-1] / plain[-1]) - 0.25) < 1e-12
    assert attention.rotary_magnitude(1) == 1 and attention.rotary_magnitude(8) > 1.2


def test_refusals():
    q = _values(1, 3, 2, 64)
    plan = attention.Rotary(attention.rotary_frequencies(64))
    for bad, error, match in (
            (lambda: attention.apply_rotary(plan, q.cpu()), ValueError, "GPU"),
            (lambda: attention.apply_rotary(plan, q.double()), TypeError, "bfloat16"),
            (lambda: attention.apply_rotary(plan, q[0]), ValueError, "4 dimensions"),
            (lambda: attention.apply_rotary(plan, q[..., :32]), ValueError, "channels"),
            (lambda: attention.apply_rotary(plan, q, q.float()), TypeError, "one type"),
            (lambda: attention.apply_rotary(plan, q, q[:, :2]), ValueError, "agree"),
            (lambda: attention.apply_rotary(plan, q, positions=1.5), TypeError, "positions"),
            (lambda: attention.apply_rotary(plan, q, positions=torch.zeros(2, device=DEV)),
             TypeError, "positions"),
            (lambda: attention.apply_rotary(
                plan, q, positions=torch.zeros(2, dtype=torch.int32, device=DEV)), ValueError,
             "positions"),
            (lambda: attention.apply_rotary("plan", q), TypeError, "plan"),
            (lambda: attention.Rotary([1.0, float("inf")]), ValueError, "finite"),
            (lambda: attention.Rotary([]), ValueError, "frequencies"),
            (lambda: attention.rotary_frequencies(7), ValueError, "even"),
            (lambda: attention.rotary_frequencies(8, scaling="other"), ValueError, "scaling")):
        with pytest.raises(error, match=match):
            bad()


@pytest.mark.parametrize("start", [2 ** 31, -2 ** 31, 1234567890])
def test_far_positions_have_exact_angles(start):
    """Against angles reduced in whole numbers."""
    tokens, dim = 4, 64
    x = _values(1, tokens, 2, dim, dtype=FP32)
    frequencies = attention.rotary_frequencies(dim)
    got = attention.apply_rotary(attention.Rotary(frequencies), x, positions=start)
    turn = 2 * Fraction("3.14159265358979323846264338327950288419716939937510582097494")
    for t in range(tokens):
        angles = [float((Fraction(f) * (start + t)) % turn) for f in frequencies.tolist()]
        _near(got[:, t:t + 1], x[:, t:t + 1], torch.ones(1, 1), angles, FP32)
    with pytest.raises(ValueError, match="positions"):
        attention.apply_rotary(attention.Rotary(frequencies), x, positions=2 ** 31 + 1)


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dim,turned", [(256, 256), (10, 6)])
def test_as_many_heads_as_are_allowed(dim, turned, interleaved):
    """4096 query and key heads: more units per token than 2^16."""
    frequencies = attention.rotary_frequencies(turned)
    plan = attention.Rotary(frequencies, interleaved=interleaved)
    q, k = (_values(1, 2, 4096, dim, dtype=FP32, seed=s) for s in (0, 1))
    at = _positions(1, 2, 3)
    for x, got in zip((q, k), attention.apply_rotary(plan, q, k, positions=3)):
        _near(got, x, at, frequencies, FP32, interleaved=interleaved)
    caches = [torch.zeros(1, 5, 4096, dim, device=DEV) for _ in range(2)]
    where = torch.tensor([4], device=DEV)
    got = attention.rotary_append(plan, q[:, 0], k[:, 0], k[:, 1], *caches, where)
    one = torch.tensor([[4]])
    _near(got.unsqueeze(1), q[:, :1], one, frequencies, FP32, interleaved=interleaved)
    _near(caches[0][:, 4:], k[:, :1], one, frequencies, FP32, interleaved=interleaved)
    assert torch.equal(caches[1][:, 4], k[:, 1])
    assert not bool(caches[0][:, :4].any()) and not bool(caches[1][:, :4].any())
