"""Windowed attention of values whose products leave FP16's normal range: gradients
of training (far below one, large, of unequal rows) over thousands of keys.

The kernels round the softmax weights, the score gradients, the output that delta is
taken from and the results to the tensors' type: relative errors of `unit` each at
most, independent from element to element.  The norm of a result's error is held to
twice that of those roundings together (their root mean square is less than 0.6 of
`unit`; the rest is for FP32's steps, 2^-24 a piece)."""
from __future__ import annotations

import attention_oracle as oracle
import pytest
import test_gpu_attention as plain
import torch

from losslessly_compressed_tensors_amd.components import attention
from losslessly_compressed_tensors_amd.kernels import attention as kernels

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF16, FP16 = torch.bfloat16, torch.float16


def _values(*shape, seed=0):
    return torch.randn(*shape, generator=torch.Generator(DEV).manual_seed(seed), device=DEV,
                       dtype=torch.float64)


def _expected(q, k, v, grad, seen, scale):
    """{name: (exact, mean square of its roundings, element by element)}."""
    dtype, unit = q.dtype, oracle.UNIT[q.dtype]
    group = q.shape[1] // k.shape[1]
    out, p = oracle.attention(q, k, v, seen, scale)
    q, grad = q.double(), grad.double()
    kk, vv = (t.double().repeat_interleave(group, 1) for t in (k, v))
    ds = p * (grad @ vv.transpose(-1, -2) - (grad * out).sum(-1, keepdim=True))
    delta = unit ** 2 * (grad.square() @ out.square().transpose(-1, -2)).diagonal(
        dim1=-2, dim2=-1).unsqueeze(-1)

    def shared(t):
        return t.unflatten(1, (k.shape[1], group)).sum(2)

    def rounded(exact, squares):
        result = exact.to(dtype).double()
        return exact, squares + (result - exact).square()

    square = scale ** 2
    return {
        "out": rounded(out, unit ** 2 * (p.square() @ vv.square())),
        "dq": rounded(scale * (ds @ kk), square * (unit ** 2 * (ds.square() @ kk.square())
                                                   + delta * (p @ kk).square())),
        "dk": rounded(scale * shared(ds.transpose(-1, -2) @ q), square * shared(
            unit ** 2 * (ds.square().transpose(-1, -2) @ q.square())
            + p.square().transpose(-1, -2) @ (delta * q.square()))),
        "dv": rounded(shared(p.transpose(-1, -2) @ grad), shared(
            unit ** 2 * (p.square().transpose(-1, -2) @ grad.square())))}


def _check(q, k, v, grad, scale=None, **how):
    scale = q.shape[3] ** -0.5 if scale is None else scale
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    out = attention.window_attention(*leaves, scale=scale, **how)
    got = dict(zip(("out", "dq", "dk", "dv"), (out.detach(),
                                               *torch.autograd.grad(out, leaves, grad))))
    seen = oracle.sees(q.shape[2], k.shape[2], how.get("window"), how.get("sinks", 0)).to(DEV)
    for name, (exact, squares) in _expected(q, k, v, grad, seen, scale).items():
        error = (got[name].double() - exact).square()
        # All tokens, and eighths of them: late queries see the most keys.
        for part in (slice(None), *(slice(i * exact.shape[2] // 8, (i + 1) * exact.shape[2] // 8)
                                    for i in range(8))):
            far, allowed = (float(t[:, :, part].sum().sqrt()) for t in (error, squares))
            assert far <= 2 * allowed, (name, part, far / allowed)


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("size", [1.0, 1e-3, 1e-4])
def test_gradients_of_any_size_over_thousands_of_keys(size, dim, dtype):
    q, k, v, grad = (_values(1, h, 4096, dim, seed=i) for i, h in enumerate((2, 1, 1, 2)))
    _check(*(t.to(dtype) for t in (q, k, v, size * grad)))


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("dim", [64, 96])
def test_gradients_of_unequal_rows(dim, dtype):
    """The largest dS of a key, of a query, comes late and is passed several times."""
    q, k, v, grad = (_values(1, h, 2000, dim, seed=i) for i, h in enumerate((2, 1, 1, 2)))
    rising = torch.logspace(-14, 6, 2000, base=2.0, device=DEV, dtype=torch.float64).view(-1, 1)
    for values, grads in ((v, grad * rising), (v, grad * rising.flip(0)), (v * rising, grad),
                          (v * rising.flip(0), 1e-2 * grad)):
        _check(*(t.to(dtype) for t in (q, k, values, grads)), window=1500, sinks=3)


@pytest.mark.parametrize("dim", [64, 128])
def test_large_gradients(dim):
    """dS beyond FP16's largest number."""
    q, k, v, grad = (_values(1, 2, 700, dim, seed=i) for i in range(4))
    _check(*(t.to(FP16) for t in (q, k, v, 5e3 * grad)), scale=0.02)


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("sink", [0, 39_999])
def test_many_small_weights_beside_a_large_one(sink, dtype, monkeypatch):
    """40000 keys of which one outscores the others by 18: their weights are e^-18 =
    2^-26 of its own, and the result is theirs alone, its value being 0."""
    for name in ("forward_splits", "decode_splits"):     # all weights beside the largest
        monkeypatch.setattr(kernels, name, lambda *a: 1)
    keys, dim, gap = 40_000, 64, 18.0
    q = torch.ones(1, 1, 1, dim, dtype=dtype, device=DEV)
    k = torch.zeros(1, 1, keys, dim, dtype=dtype, device=DEV)
    k[:, :, sink] = gap / dim
    v = torch.ones(1, 1, keys, dim, dtype=dtype, device=DEV)
    v[:, :, sink] = 0.0
    exact, _ = oracle.attention(q, k, v, oracle.sees(1, keys).to(DEV), 1.0)
    # Each weight's rounding, of FP16's least step where it is held 2^7 larger than its
    # share of the largest; the sums' FP32 steps; the result's rounding.
    unit = oracle.UNIT[dtype]
    bound = (2 * unit + keys * oracle.STEP) * exact + (keys * 2.0 ** -32 if dtype == FP16 else 0.0)
    lengths = torch.tensor([keys], device=DEV)
    got = attention.window_attention(q, k, v, scale=1.0)
    one = attention.decode_attention(q[:, :, 0], k.transpose(1, 2), v.transpose(1, 2), lengths,
                                     scale=1.0)
    for value in (got[:, :, 0], one):
        assert bool(((value.double() - exact[:, :, 0]).abs() <= bound[:, :, 0]).all()), (
            float(value.flatten()[0]), float(exact.flatten()[0]))


@pytest.mark.parametrize("dim,splits", [(64, None), (128, None), (64, 3)])
@pytest.mark.parametrize("where", ["v", "k", "q", "grad"])
@pytest.mark.parametrize("value", [float("nan"), float("inf")])
def test_infinities_in_fp16(where, value, dim, splits, monkeypatch):
    """The power of two that dS is held at follows finite values alone."""
    monkeypatch.setattr(plain._inputs, "__defaults__", (FP16,))
    plain.test_infinities_reach_only_what_sees_them(where, value, dim, splits, monkeypatch)


def test_padding_in_fp16(monkeypatch):
    monkeypatch.setattr(plain._inputs, "__defaults__", (FP16,))
    plain.test_padding_may_hold_anything()
