"""Windowed attention, its gradients and its single-token form against the
definitions in 64 bits (``attention_oracle``), at the sizes and masks where tiles,
splits and empty rows can go wrong."""
from __future__ import annotations

import attention_oracle as oracle
import pytest
import torch

from losslessly_compressed_tensors_amd.components import attention
from losslessly_compressed_tensors_amd.kernels import attention as kernels

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF16, FP16 = torch.bfloat16, torch.float16


def _values(*shape, dtype=BF16, seed=0):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(dtype).to(DEV)


def _inputs(batch, heads, kv_heads, queries, keys, dim, dtype=BF16):
    """BHTD views of BTHD storage: q, k, v, grad."""
    return [_values(batch, t, h, dim, dtype=dtype, seed=i).transpose(1, 2)
            for i, (t, h) in enumerate(((queries, heads), (keys, kv_heads), (keys, kv_heads),
                                        (queries, heads)))]


def _run(q, k, v, grad, **how):
    q, k, v = (t.detach().requires_grad_() for t in (q, k, v))
    out = attention.window_attention(q, k, v, **how)
    return dict(zip(("out", "dq", "dk", "dv"),
                    (out.detach(), *torch.autograd.grad(out, (q, k, v), grad))))


def _check(got, expected):
    for name, (exact, bound) in expected.items():
        value = got[name]
        assert value.shape == exact.shape, name
        far = (value.double() - exact).abs() - bound
        assert bool((far <= 0).all()), (name, float(far.max()), int((far > 0).sum()))


# batch, heads, key heads, queries, keys, channels, window, sinks, lengths
CASES = [
    (1, 1, 1, 1, 1, 8, None, 0, None),
    (2, 2, 2, 2, 2, 64, None, 0, None),
    (1, 2, 1, 31, 31, 32, 2, 0, None),
    (2, 4, 2, 130, 130, 64, 33, 3, None),
    (1, 3, 3, 128, 128, 64, None, 0, None),
    (1, 2, 1, 129, 129, 128, 64, 64, None),
    (1, 6, 2, 257, 257, 80, 100, 1, None),
    (1, 2, 2, 300, 300, 40, 1, 200, None),        # sinks past a key block, window of one
    (1, 2, 1, 400, 400, 96, 5, 1000, None),       # more sinks than keys
    (2, 2, 1, 65, 200, 128, None, 0, None),       # a chunk of new tokens
    (2, 4, 1, 70, 333, 64, 90, 7, None),
    (1, 2, 1, 200, 65, 64, 40, 2, None),          # queries before the first key see nothing
    (4, 2, 1, 150, 150, 96, 50, 2, [0, 1, 77, 150]),
    (3, 4, 4, 129, 260, 64, None, 0, [260, 131, 5]),
    (1, 1, 1, 16, 1500, 64, None, 0, None),       # keys shared among workgroups
    (1, 8, 2, 3, 900, 128, 600, 4, [850]),
    (1, 2, 1, 1100, 1100, 32, 130, 5, None),      # the sinks' queries shared among workgroups
]


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("case", CASES, ids=lambda c: "x".join(map(str, c[:8])))
def test_attention_and_gradients(case, dtype):
    batch, heads, kv_heads, queries, keys, dim, window, sinks, lengths = case
    q, k, v, grad = _inputs(batch, heads, kv_heads, queries, keys, dim, dtype)
    scale = dim ** -0.5
    seen = oracle.sees(queries, keys, window, sinks, lengths, batch).to(DEV)
    sized = None if lengths is None else torch.tensor(lengths, dtype=torch.int32, device=DEV)
    got = _run(q, k, v, grad, window=window, sinks=sinks, lengths=sized)
    _check(got, oracle.attention_with_bounds(q, k, v, seen, scale, grad))
    empty = ~seen.any(-1).expand(batch, heads, queries)
    assert bool((got["out"][empty] == 0).all()) and bool((got["dq"][empty] == 0).all())
    assert torch.equal(attention.window_attention(q, k, v, window=window, sinks=sinks,
                                                  lengths=sized), got["out"])


@pytest.mark.parametrize("splits", [1, 2, 5, 64])
def test_the_number_of_parts_changes_rounding_only(splits, monkeypatch):
    monkeypatch.setattr(kernels, "forward_splits", lambda *a: splits)
    monkeypatch.setattr(kernels, "backward_splits", lambda *a: (splits, min(64, 2 * splits)))
    q, k, v, grad = _inputs(2, 4, 2, 300, 700, 64)
    seen = oracle.sees(300, 700, 257, 130, None, 2).to(DEV)
    got = _run(q, k, v, grad, window=257, sinks=130, scale=0.2)
    _check(got, oracle.attention_with_bounds(q, k, v, seen, 0.2, grad))
    again = _run(q, k, v, grad, window=257, sinks=130, scale=0.2)
    assert all(torch.equal(got[n], again[n]) for n in got)


def test_gradients_against_differences():
    """Along random directions, the 64-bit definition's central differences."""
    q, k, v, grad = _inputs(1, 4, 2, 140, 140, 64)
    seen = oracle.sees(140, 140, 50, 3).to(DEV)
    got = _run(q, k, v, grad, window=50, sinks=3, scale=0.12)
    expected = oracle.attention_with_bounds(q, k, v, seen, 0.12, grad)
    step = 1e-5
    for at, name in enumerate(("dq", "dk", "dv")):
        along = torch.randn((q, k, v)[at].shape, device=DEV, dtype=torch.float64,
                            generator=torch.Generator(DEV).manual_seed(at))
        sides = []
        for sign in (1, -1):
            inputs = [t.double() for t in (q, k, v)]
            inputs[at] = inputs[at] + sign * step * along
            out, _ = oracle.attention(*inputs, seen, 0.12)
            sides.append((out * grad.double()).sum())
        difference = (sides[0] - sides[1]) / (2 * step)
        allowed = (expected[name][1] * along.abs()).sum() + 1e-6 * difference.abs() + 1e-6
        assert abs((got[name].double() * along).sum() - difference) <= allowed


def test_strides_and_broadcast_inputs():
    """Slices of one projection, head-major storage, an odd offset, shared tokens,
    a broadcast gradient: the results of plain copies."""
    both = _values(2, 150, 8, 64)
    q, k, v = (t.transpose(1, 2) for t in both.split((4, 2, 2), dim=2))
    grad = _values(2, 4, 150, 64, seed=5)
    want = _run(*(t.contiguous() for t in (q, k, v, grad)), window=40, sinks=2)
    got = _run(q, k, v, grad, window=40, sinks=2)
    assert all(torch.equal(got[n], want[n]) for n in want)

    flat = torch.zeros(2 * 4 * 150 * 64 + 3, dtype=BF16, device=DEV)
    odd = flat[3:].view(2, 4, 150, 64)
    odd.copy_(q)
    got = _run(odd, k, v, grad, window=40, sinks=2)
    assert all(torch.equal(got[n], want[n]) for n in want)

    last = _values(2, 4, 64, 150, seed=9).transpose(2, 3)       # channels not adjacent
    got = _run(last, k, v, grad, window=40, sinks=2)
    assert all(torch.equal(got[n], w) for n, w in
               _run(last.contiguous(), k, v, grad, window=40, sinks=2).items())

    one = _values(2, 2, 1, 64, seed=6)
    broad = one.expand(2, 2, 150, 64)
    leaf = one.clone().requires_grad_()
    out = attention.window_attention(q, leaf.expand(2, 2, 150, 64), v, window=40)
    assert torch.equal(out, attention.window_attention(q, broad.contiguous(), v, window=40))
    out.sum().backward()                                        # the gradient is broadcast too
    plain = _run(q, broad.contiguous(), v, torch.ones_like(q), window=40)
    bound = 150 * 2.0 ** -8 * plain["dk"].double().abs().sum(2, keepdim=True) + 1e-6
    assert bool(((leaf.grad.double() - plain["dk"].double().sum(2, keepdim=True)).abs()
                 <= bound).all())


def test_padding_may_hold_anything():
    """NaN and infinities past the sequences' lengths reach nothing."""
    q, k, v, grad = _inputs(2, 4, 2, 200, 200, 64)
    lengths = torch.tensor([131, 64], device=DEV)
    want = _run(q, k, v, grad, window=60, sinks=3, lengths=lengths)
    for t, value in ((q, float("nan")), (k, float("inf")), (v, float("nan")),
                     (grad, float("-inf"))):
        for b, n in enumerate((131, 64)):
            t[b, :, n:] = value
    got = _run(q, k, v, grad, window=60, sinks=3, lengths=lengths)
    assert all(torch.equal(got[n], want[n]) for n in want)
    assert all(bool(got[n].isfinite().all()) for n in got)


def test_large_scores():
    """Scores of a thousand: the running maximum moves, most weights vanish."""
    q, k, v, grad = _inputs(1, 2, 2, 190, 190, 64)
    q, k = q * 20, k * 20
    seen = oracle.sees(190, 190, 100, 1).to(DEV)
    got = _run(q, k, v, grad, window=100, sinks=1, scale=0.125)
    _check(got, oracle.attention_with_bounds(q, k, v, seen, 0.125, grad))


def test_nothing_to_attend():
    q = _values(2, 4, 0, 64)
    kv = _values(2, 2, 5, 64)
    assert attention.window_attention(q, kv, kv).shape == (2, 4, 0, 64)
    q, none = _values(2, 4, 3, 64).requires_grad_(), _values(2, 2, 0, 64)
    out = attention.window_attention(q, none, none)
    assert bool((out == 0).all())
    out.sum().backward()
    assert bool((q.grad == 0).all())


# batch, heads, key heads, capacity, channels, window, sinks, lengths
DECODE = [
    (1, 1, 1, 1, 8, None, 0, [1]),
    (1, 12, 12, 257, 64, None, 0, [257]),
    (4, 8, 2, 300, 128, None, 0, [0, 1, 33, 300]),
    (3, 8, 1, 1000, 80, 200, 5, [1000, 204, 3]),
    (2, 20, 1, 500, 64, 64, 0, [500, 64]),          # more than 16 queries per key head
    (2, 32, 2, 700, 96, 31, 40, [700, 71]),
    (1, 4, 2, 5000, 32, None, 0, [4999]),
    (1, 2, 2, 130, 128, 1, 0, [129]),
    (2, 4, 4, 64, 64, 8, 300, [64, 40]),            # all sinks
    (1, 3, 3, 50, 64, None, 0, [80]),               # a length past the capacity counts as it
]


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("case", DECODE, ids=lambda c: "x".join(map(str, c[:7])))
def test_decode(case, dtype):
    batch, heads, kv_heads, capacity, dim, window, sinks, lengths = case
    q = _values(batch, heads, dim, dtype=dtype)
    k, v = (_values(batch, capacity, kv_heads, dim, dtype=dtype, seed=s) for s in (1, 2))
    sized = torch.tensor(lengths, dtype=torch.int32, device=DEV)
    live = [min(n, capacity) for n in lengths]
    for b, n in enumerate(live):        # what lies past a sequence may be anything
        k[b, n:], v[b, n:] = float("nan"), float("inf")
        if window is not None:          # and so may what the window has left
            k[b, sinks:max(sinks, n - window)] = float("nan")
            v[b, sinks:max(sinks, n - window)] = float("inf")
    got = attention.decode_attention(q, k, v, sized, window=window, sinks=sinks)
    assert got.shape == q.shape
    for b, n in enumerate(live):
        if n == 0:
            assert bool((got[b] == 0).all())
            continue
        seen = oracle.sees(1, n, window, sinks).to(DEV)
        kk, vv = (t[b:b + 1, :n].transpose(1, 2) for t in (k, v))
        kk, vv = (torch.where(seen[..., 0, :, None], t, 0) for t in (kk, vv))
        _check({"out": got[b:b + 1].unsqueeze(2)},
               oracle.attention_with_bounds(q[b:b + 1].unsqueeze(2), kk, vv, seen, dim ** -0.5))


@pytest.mark.parametrize("splits", [1, 3, 64])
def test_decode_parts_and_head_major_caches(splits, monkeypatch):
    monkeypatch.setattr(kernels, "decode_splits", lambda *a: splits)
    q = _values(2, 8, 64)
    k, v = (_values(2, 2, 600, 64, seed=s).transpose(1, 2) for s in (1, 2))
    lengths = torch.tensor([600, 17], device=DEV)
    got = attention.decode_attention(q, k, v, lengths, window=300, sinks=9, scale=0.3)
    for b, n in enumerate((600, 17)):
        _check({"out": got[b:b + 1].unsqueeze(2)}, oracle.attention_with_bounds(
            q[b:b + 1].unsqueeze(2), *(t[b:b + 1, :n].transpose(1, 2) for t in (k, v)),
            oracle.sees(1, n, 300, 9).to(DEV), 0.3))


def test_decode_of_strided_and_misaligned_tensors():
    """Results of plain copies: a query and caches at odd addresses, channels not
    adjacent, slices of wider tensors."""
    q = _values(2, 4, 64)
    k, v = (_values(2, 90, 2, 64, seed=s) for s in (1, 2))
    lengths = torch.tensor([90, 31], device=DEV)
    want = attention.decode_attention(q, k, v, lengths, window=20, sinks=1)

    def odd(t):
        out = torch.zeros(t.numel() + 1, dtype=BF16, device=DEV)[1:].view(t.shape)
        out.copy_(t)
        return out

    def turned(t):
        return t.transpose(-1, -2).contiguous().transpose(-1, -2)

    def slice_of_wider(t):
        wide = torch.zeros(*t.shape[:-1], 72, dtype=BF16, device=DEV)
        wide[..., :64] = t
        return wide[..., :64]

    for other in (odd, turned, slice_of_wider):
        got = attention.decode_attention(other(q), other(k), other(v), lengths, window=20, sinks=1)
        assert torch.equal(got, want)


def test_decode_is_the_last_row_of_attention():
    """The cache's path and the prompt's agree within their bounds."""
    plan = attention.Rotary(attention.rotary_frequencies(64))
    cache = attention.KVCache(2, 100, 2, 64)
    q, k, v = (_values(2, 70, h, 64, seed=h) for h in (4, 2, 2))
    with torch.no_grad():
        rq, rk = cache.fill(plan, q[:, :60], k[:, :60], v[:, :60])
        assert torch.equal(cache.k[:, :60], rk) and cache.lengths.tolist() == [60, 60]
        for t in range(60, 70):
            turned = cache.append(plan, q[:, t], k[:, t], v[:, t])
            out = cache.attend(turned, window=30, sinks=2)
        all_q, all_k = attention.apply_rotary(plan, q, k)
        whole = attention.window_attention(all_q.transpose(1, 2), all_k.transpose(1, 2),
                                           v.transpose(1, 2), window=30, sinks=2)
    assert torch.equal(cache.k[:, :70], all_k) and torch.equal(cache.v[:, :70], v)
    assert torch.equal(turned, all_q[:, -1])
    bounds = oracle.attention_with_bounds(
        all_q.transpose(1, 2), all_k.transpose(1, 2), v.transpose(1, 2),
        oracle.sees(70, 70, 30, 2).to(DEV), 64 ** -0.5)["out"][1][:, :, -1]
    assert bool(((out.double() - whole[:, :, -1].double()).abs() <= 2 * bounds).all())
    with pytest.raises(ValueError, match="holds 100 tokens"):
        for _ in range(31):
            cache._grow(1)
    cache.reset()
    assert cache.lengths.tolist() == [0, 0]


def test_another_stream():
    q, k, v, grad = _inputs(1, 4, 2, 300, 300, 64)
    want = _run(q, k, v, grad, window=100, sinks=1)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        got = _run(q, k, v, grad, window=100, sinks=1)
    stream.synchronize()
    assert all(torch.equal(got[n], want[n]) for n in want)


def test_a_captured_step_replays():
    """Decode steps in a graph, lengths advancing on the device: every replay gives
    the eager result."""
    plan = attention.Rotary(attention.rotary_frequencies(64))
    q, k, v = (_values(6, 2, h, 64, seed=h) for h in (8, 2, 2))

    def step(cache, at):
        out = cache.attend(attention.rotary_append(plan, at[0], at[1], at[2], cache.k, cache.v,
                                                   cache.lengths - 1), window=4, sinks=1)
        return out

    eager, caught = attention.KVCache(2, 700, 2, 64), attention.KVCache(2, 700, 2, 64)
    at = [t[0].clone() for t in (q, k, v)]
    with torch.no_grad():
        caught.lengths.fill_(1)
        step(caught, at)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            result = step(caught, at)
        caught.lengths.fill_(0)
        for i in range(6):
            for t, new in zip(at, (q, k, v)):
                t.copy_(new[i])
            caught.lengths += 1
            eager.lengths += 1
            graph.replay()
            torch.cuda.synchronize()
            want = step(eager, [t[i] for t in (q, k, v)])
            assert torch.equal(result, want)


def test_nothing_to_see_is_zero_whatever_the_query_holds():
    q = _values(1, 2, 3, 64)
    q[0, 0, 0, 0], q[0, 1, 2, 3] = float("inf"), float("nan")
    q.requires_grad_()
    none = _values(1, 2, 0, 64)
    out = attention.window_attention(q, none, none)
    assert bool((out == 0).all())
    out.sum().backward()
    assert bool((q.grad == 0).all())


def test_lengths_past_32_bits_count_as_the_capacity():
    q, cache = _values(3, 4, 64), _values(3, 20, 2, 64, seed=1)
    got = attention.decode_attention(
        q, cache, cache, torch.tensor([2 ** 32 + 5, 20, -2 ** 32 + 20], device=DEV))
    want = attention.decode_attention(q, cache, cache, torch.tensor([20, 20, 0], device=DEV))
    assert torch.equal(got, want)
    # A place past the cache is not written.
    plan = attention.Rotary(attention.rotary_frequencies(64))
    before = cache.clone()
    attention.rotary_append(plan, q, q[:, :2], q[:, 2:], cache, cache.clone(),
                            torch.tensor([2 ** 32, 2 ** 33 + 1, -2 ** 32], device=DEV))
    assert torch.equal(cache, before)


def test_a_refused_call_leaves_the_cache_as_it_was():
    plan = attention.Rotary(attention.rotary_frequencies(64))
    cache = attention.KVCache(2, 4, 2, 64)
    q, k = _values(2, 3, 4, 64), _values(2, 3, 2, 64)
    for bad, error, match in (
            (lambda: cache.fill(plan, q, k, k[:1]), ValueError, "cache's heads"),
            (lambda: cache.fill(plan, q, k[:, :, :1], k[:, :, :1]), ValueError, "cache's heads"),
            (lambda: cache.fill(plan, q, k, k.half()), TypeError, "one type"),
            (lambda: cache.fill(plan, q.half(), k, k), TypeError, "one type"),
            (lambda: cache.fill(plan, q, k.clone().requires_grad_(), k), ValueError, "gradient"),
            (lambda: cache.fill(plan, *[torch.cat([t, t], 1) for t in (q, k, k)]), ValueError,
             "holds 4 tokens"),
            (lambda: cache.append(plan, q[:, 0], k[:, 0], k[:1, 0]), ValueError, "agree"),
            (lambda: attention.KVCache(1, 4, 0, 64), ValueError, "kv_heads"),
            (lambda: attention.KVCache(1, 4, 2.0, 64), TypeError, "kv_heads")):
        with pytest.raises(error, match=match):
            bad()
    cache.fill(plan, q, k, k)
    cache.append(plan, q[:, 0], k[:, 0], k[:, 0])
    assert cache.lengths.tolist() == [4, 4]
    with pytest.raises(ValueError, match="holds 4 tokens"):
        cache.append(plan, q[:, 0], k[:, 0], k[:, 0])
    assert cache.lengths.tolist() == [4, 4]


def test_append_writes_to_its_caches_alone():
    plan = attention.Rotary(attention.rotary_frequencies(64))
    q, k = _values(2, 4, 64), _values(2, 2, 64)
    cache, at = _values(2, 5, 2, 64), torch.zeros(2, dtype=torch.int32, device=DEV)
    for shared in (cache[:1].expand(2, 5, 2, 64), cache[:, :1].expand(2, 5, 2, 64)):
        with pytest.raises(ValueError, match="expanded"):
            attention.rotary_append(plan, q, k, k, shared, cache, at)
    # A graph that has saved a cache refuses to go on with other values.
    weights = torch.ones(64, dtype=BF16, device=DEV, requires_grad=True)
    out = (cache * weights).sum()
    attention.rotary_append(plan, q, k, k, cache, cache.clone(), at)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        out.backward()


def test_refusals():
    q, k = _values(1, 4, 5, 64), _values(1, 2, 5, 64)
    call = attention.window_attention
    for bad, error, match in (
            (lambda: call(q.cpu(), k, k), ValueError, "GPU"),
            (lambda: call(q.float(), k, k), TypeError, "bfloat16"),
            (lambda: call(q, k.half(), k), TypeError, "one type"),
            (lambda: call(q[0], k, k), ValueError, "4 dimensions"),
            (lambda: call(q, k, k[:, :, :4]), ValueError, "agree"),
            (lambda: call(_values(1, 3, 5, 64), k, k), ValueError, "multiple"),
            (lambda: call(*[_values(1, 2, 5, 12)] * 3), ValueError, "channels"),
            (lambda: call(*[_values(1, 2, 5, 136)] * 3), ValueError, "channels"),
            (lambda: call(q, k, k, window=0), ValueError, "window"),
            (lambda: call(q, k, k, window=2.0), TypeError, "window"),
            (lambda: call(q, k, k, sinks=-1), ValueError, "sinks"),
            (lambda: call(q, k, k, scale=0.0), ValueError, "scale"),
            (lambda: call(q, k, k, scale=float("nan")), ValueError, "scale"),
            (lambda: call(q, k, k, lengths=torch.ones(2, dtype=torch.int32, device=DEV)),
             ValueError, "lengths"),
            (lambda: call(q, k, k, lengths=torch.ones(1, device=DEV)), TypeError, "lengths"),
            (lambda: call(q, k, k, lengths=torch.ones(1, dtype=torch.int32)), ValueError,
             "lengths")):
        with pytest.raises(error, match=match):
            bad()
    cache = _values(1, 9, 2, 64)
    one = torch.ones(1, dtype=torch.int32, device=DEV)
    query = _values(1, 4, 64)
    decode = attention.decode_attention
    for bad, error, match in (
            (lambda: decode(q, cache, cache, one), ValueError, "3 dimensions"),
            (lambda: decode(query, cache, cache[:, :8], one), ValueError, "agree"),
            (lambda: decode(query, cache, cache, None), TypeError, "lengths"),
            (lambda: decode(query.clone().requires_grad_(), cache, cache, one), ValueError,
             "gradient"),
            (lambda: decode(_values(1, 3, 64), cache, cache, one), ValueError, "multiple")):
        with pytest.raises(error, match=match):
            bad()
    leaf = q.clone().requires_grad_()
    grad, = torch.autograd.grad(call(leaf, k, k).float().sum(), leaf, create_graph=True)
    with pytest.raises(RuntimeError):
        grad.sum().backward()


@pytest.mark.parametrize("dim,splits", [(64, None), (128, None), (64, 3)])
@pytest.mark.parametrize("where", ["v", "k", "q", "grad"])
@pytest.mark.parametrize("value", [float("nan"), float("inf")])
def test_infinities_reach_only_what_sees_them(where, value, dim, splits, monkeypatch):
    """One token of one tensor is not finite: results that it has no part in keep
    their bounds, whatever tiles they share with it; those that it has are not
    finite."""
    if splits is not None:
        monkeypatch.setattr(kernels, "forward_splits", lambda *a: splits)
        monkeypatch.setattr(kernels, "backward_splits", lambda *a: (splits, splits))
    tokens, window, sinks, at = 260, 40, 2, 100
    clean = dict(zip("qkv", _inputs(1, 2, 1, tokens, tokens, dim)[:3]),
                 grad=_inputs(1, 2, 1, tokens, tokens, dim)[3])
    seen = oracle.sees(tokens, tokens, window, sinks).to(DEV)
    pairs = seen[0, 0]
    poisoned = {n: t.clone() for n, t in clean.items()}
    poisoned[where][:, :, at] = value
    got = _run(*(poisoned[n] for n in ("q", "k", "v", "grad")), window=window, sinks=sinks)
    # Rows and keys that the token has a part in, and the results without it.
    if where in "kv":
        rows = pairs[:, at]
        without = seen.clone()
        without[..., at] = False
    else:
        rows = torch.arange(tokens, device=DEV) == at
        without = seen.clone()
        without[..., at, :] = False
    keys = pairs[rows].any(0)
    for name, (exact, bound) in oracle.attention_with_bounds(
            *(clean[n] for n in "qkv"), without, dim ** -0.5, clean["grad"]).items():
        # The output does not depend on the gradient that comes back.
        if name == "out" and where == "grad":
            continue
        clear = ~(rows if name in ("out", "dq") else keys)
        far = (got[name].double() - exact).abs() - bound
        assert bool((far[:, :, clear] <= 0).all()), name
    if where != "grad":
        assert not bool(got["out"][:, :, rows].isfinite().all(-1).any()) or value == float("inf")
    assert bool(got["dq"][:, :, ~rows].isfinite().all())
    assert bool(got["dk"][:, :, ~keys].isfinite().all())


def test_offsets_past_32_bits():
    """A cache of over 2^31 bytes per tensor: its last tokens through the append,
    the single-token and the chunk form, and the chunk's gradients."""
    tokens, kv_heads, dim, window, sinks = 1_100_000, 8, 128, 300, 3
    assert tokens * kv_heads * dim * 2 > 2 ** 31
    caches = [torch.zeros(1, tokens, kv_heads, dim, dtype=BF16, device=DEV) for _ in range(2)]
    near = 1000
    for i, cache in enumerate(caches):
        cache[:, :sinks] = _values(1, sinks, kv_heads, dim, seed=10 + i)
        cache[:, -near:] = _values(1, near, kv_heads, dim, seed=20 + i)
    plan = attention.Rotary(attention.rotary_frequencies(dim))
    q, k, v = (_values(1, h, dim, seed=h) for h in (16, 8, 8))
    at = torch.tensor([tokens - 1], dtype=torch.int32, device=DEV)
    q = attention.rotary_append(plan, q, k, v, *caches, at)
    assert torch.equal(caches[1][:, -1], v)
    assert torch.equal(caches[0][:, -1:], attention.apply_rotary(plan, k.unsqueeze(1),
                                                                 positions=at))
    got = attention.decode_attention(q, *caches, at + 1, window=window, sinks=sinks)
    # The same keys next to each other: sinks, then the last 1000.
    small = [torch.cat([c[:, :sinks], c[:, -near:]], 1).transpose(1, 2) for c in caches]
    seen = oracle.sees(1, sinks + near, window, sinks).to(DEV)
    _check({"out": got.unsqueeze(2)},
           oracle.attention_with_bounds(q.unsqueeze(2), *small, seen, dim ** -0.5))

    queries = 70
    chunk, grad = (_values(1, queries, 16, dim, seed=s).transpose(1, 2) for s in (31, 32))
    result = _run(chunk, *(c.transpose(1, 2) for c in caches), grad, window=window, sinks=sinks)
    seen = oracle.sees(queries, sinks + near, window, sinks).to(DEV)
    for name in ("dk", "dv"):
        full = result[name]
        assert bool((full[:, :, sinks:-near] == 0).all())
        result[name] = torch.cat([full[:, :, :sinks], full[:, :, -near:]], 2)
    _check(result, oracle.attention_with_bounds(chunk, *small, seen, dim ** -0.5, grad))


@pytest.mark.parametrize("splits,sink_splits", [(1, 5), (3, 1), (3, 5), (1, 1)])
@pytest.mark.parametrize("dim", [64, 128])
def test_parts_of_one_kind_of_key_block(dim, splits, sink_splits, monkeypatch):
    """Blocks with sinks in parts and the others whole, the other way round, both:
    the parts fill the workspace that is asked for, and no more."""
    sizes = []
    monkeypatch.setattr(kernels, "backward_splits", lambda *a: (splits, sink_splits))
    plain = kernels._workspace

    def guarded(q, floats):
        sizes.append(floats)
        if not floats:
            return plain(q, floats)
        memory = torch.full((floats + 1024,), float("nan"), device=DEV)
        guarded.memory = memory
        return memory, memory.data_ptr()

    q, k, v, grad = _inputs(2, 4, 2, 900, 900, dim)
    seen = oracle.sees(900, 900, 100, 300, None, 2).to(DEV)
    out, lse = kernels.attention_forward(q, k, v, 100, 300, 0.1, None, True)
    monkeypatch.setattr(kernels, "_workspace", guarded)
    got = dict(zip(("out", "dq", "dk", "dv"), (out, *kernels.attention_backward(
        grad, q, k, v, out, lse, 100, 300, 0.1, None))))
    torch.cuda.synchronize()
    _check(got, oracle.attention_with_bounds(q, k, v, seen, 0.1, grad))
    if splits == sink_splits == 1:
        assert sizes == [0]
    else:
        floats, = sizes
        assert bool(guarded.memory[floats:].isnan().all())
        # Every part's keys that exist are written: the last block's others are not.
        assert int(guarded.memory[:floats].isnan().sum()) <= floats // 2


def test_gradients_of_a_sum_of_attention_are_no_constants():
    """An incoming gradient of ones needs no gradient: a second derivative is refused, not left
    out."""
    for at in range(3):
        leaves = [_values(1, 2, 9, 64).requires_grad_(i == at) for i in range(3)]
        out = attention.window_attention(*leaves, window=4).float().sum()
        plain, = torch.autograd.grad(out, leaves[at], retain_graph=True)
        grad, = torch.autograd.grad(out, leaves[at], create_graph=True)
        assert torch.equal(grad, plain)
        with pytest.raises(RuntimeError, match="differentiated once only"):
            (out + grad.float().square().sum()).backward()
