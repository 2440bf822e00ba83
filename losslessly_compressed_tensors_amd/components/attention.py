"""Rotary positions, attention with a sliding window and sinks, and the cache
that single-token attention reads.

The reference's trainer computes its rotary embedding in eager steps and calls
the library's causal attention (``examples/nanogpt/train_gpt_lct.py:150-205``,
``LCT/components/layers.py:225-305``); it has no window, no cache and no form for
single tokens.  Here each is a kernel of its own:

* :class:`Rotary` (the plan) with :func:`apply_rotary` (differentiable) and
  :func:`rotary_append` (a new token's rotation and its way into the caches);
* :func:`window_attention` (differentiable): every query sees the last ``window``
  keys up to its own and the first ``sinks`` keys;
* :func:`decode_attention`: one query per sequence over its cache;
* :class:`KVCache`: both caches and the sequences' lengths.

All take GPU tensors, launch on the current stream and never synchronise.
``components/layers.py``'s ``WindowAttention`` is the training layer that keeps
what backward needs compressed.
"""
from __future__ import annotations

import math
import numbers
from fractions import Fraction

import torch
from torch import Tensor
from torch.autograd.function import once_differentiable

from ..kernels import attention as kernels

__all__ = ["Rotary", "rotary_frequencies", "rotary_magnitude", "trainer_frequencies",
           "apply_rotary", "rotary_append", "window_attention", "decode_attention", "KVCache"]


def _whole(value, name: str, least: int, most: int) -> int:
    if isinstance(value, bool) or not isinstance(value, numbers.Integral):
        raise TypeError(f"{name} must be an integer")
    if not least <= value <= most:
        raise ValueError(f"{name} must lie between {least} and {most}, got {value}")
    return int(value)


_PLAIN = (Tensor, torch.nn.Parameter)
_wrapped = torch._C._functorch.is_functorch_wrapped_tensor


def _check_tensor(t, name: str, ndim: int, dtypes) -> None:
    if type(t) not in _PLAIN or _wrapped(t) or t.is_neg():
        raise TypeError(f"{name} must be a plain torch.Tensor, got {type(t).__name__}")
    if not t.is_cuda:
        raise ValueError(f"{name} must be a GPU tensor")
    if t.dtype not in dtypes:
        raise TypeError(f"{name} must be one of {', '.join(map(str, dtypes))}, got {t.dtype}")
    if t.ndim != ndim:
        raise ValueError(f"{name} must have {ndim} dimensions, got {t.ndim}")


def _check_like(t, name: str, other: Tensor, ndim: int) -> None:
    """``t`` against ``other``, q or x, which has been checked."""
    if type(t) not in _PLAIN or _wrapped(t) or t.is_neg():
        raise TypeError(f"{name} must be a plain torch.Tensor, got {type(t).__name__}")
    if t.device != other.device:
        raise ValueError(f"all tensors must be on {other.device}, {name} is on {t.device}")
    if t.dtype != other.dtype:
        raise TypeError(f"all tensors must have one type, {other.dtype}: {name} has {t.dtype}")
    if t.ndim != ndim:
        raise ValueError(f"{name} must have {ndim} dimensions, got {t.ndim}")


def _recorded(*tensors) -> bool:
    """Whether autograd has to see the call."""
    if not torch.is_grad_enabled():
        return False
    for t in tensors:
        if t is not None and t.requires_grad:
            return True
    return False


def _check_memory(t, name: str) -> None:
    """Tensors that the kernels may do without: an address of zero, which those
    without memory have, would mean that there is none."""
    if not isinstance(t, Tensor):
        raise TypeError(f"{name} must be a torch.Tensor")
    if type(t) not in _PLAIN or _wrapped(t) or t._is_zerotensor():
        raise TypeError(f"{name} must be a plain torch.Tensor")


def _indices(t, name: str, shapes, device) -> Tensor:
    """An index tensor as INT32 of one of ``shapes``."""
    _check_memory(t, name)
    if t.dtype not in (torch.int32, torch.int64):
        raise TypeError(f"{name} must be int32 or int64, got {t.dtype}")
    if tuple(t.shape) not in shapes:
        raise ValueError(f"{name} must have shape {' or '.join(map(str, shapes))}, "
                         f"got {tuple(t.shape)}")
    if t.device != device:
        raise ValueError(f"{name} must be on {device}")
    # Not modulo 2^32: a length or place that INT32 does not hold is past the end.
    return t if t.dtype == torch.int32 else t.clamp(-2 ** 31, 2 ** 31 - 1).to(torch.int32)


# ---- rotary positions


def rotary_frequencies(dim: int, base: float = 10000.0, *, scaling: str | None = None,
                       factor: float = 1.0, trained_length: int = 4096, slow_turns: float = 1.0,
                       fast_turns: float = 32.0) -> Tensor:
    """Radians per position of ``dim / 2`` pairs, ``base ** (-2 i / dim)``, in FP64.

    ``scaling`` stretches them for contexts ``factor`` times those of training:
    ``"linear"`` divides all by ``factor``; ``"base"`` raises the base so that the
    slowest pair is divided by it and the fastest kept; ``"ramp"`` divides the
    pairs that turn at most ``slow_turns`` times in ``trained_length`` positions,
    keeps those of at least ``fast_turns`` and goes linearly between
    (``rotary_magnitude`` belongs to it)."""
    dim = _whole(dim, "dim", 2, kernels.MAX_ROTARY_DIM)
    if dim % 2:
        raise ValueError("dim must be even")
    if not (math.isfinite(base) and base > 0) or not (math.isfinite(factor) and factor >= 1):
        raise ValueError("base must be positive and factor at least 1")
    index = torch.arange(dim // 2, dtype=torch.float64)
    if scaling == "base" and dim > 2:
        base = base * factor ** (dim / (dim - 2))
    plain = float(base) ** (-2.0 * index / dim)
    if scaling is None or scaling == "base":
        return plain
    if scaling == "linear":
        return plain / factor
    if scaling == "ramp":
        if not fast_turns > slow_turns or not trained_length > 0:
            raise ValueError("fast_turns must exceed slow_turns, and trained_length 0")
        turns = trained_length * plain / (2 * math.pi)
        keep = ((turns - slow_turns) / (fast_turns - slow_turns)).clamp(0, 1)
        return plain * (keep + (1 - keep) / factor)
    raise ValueError(f"unknown scaling {scaling!r}")


def rotary_magnitude(factor: float) -> float:
    """What ``"ramp"`` multiplies queries and keys by: 0.1 ln(factor) + 1."""
    return 0.1 * math.log(factor) + 1.0 if factor > 1 else 1.0


def trainer_frequencies(head_dim: int) -> Tensor:
    """The trainer's (``train_gpt_lct.py:150-165``): 1 to 1/1024 for the first
    half of the pairs, the others not turned, the other sense of rotation."""
    quarter = _whole(head_dim, "head_dim", 4, kernels.MAX_ROTARY_DIM) // 4
    live = (1 / 1024) ** torch.linspace(0, 1, steps=quarter, dtype=torch.float64)
    return torch.cat([-live, live.new_zeros(head_dim // 2 - quarter)])


class Rotary:
    """The plan of a rotation: ``frequencies`` (radians per position, one per
    pair), the layout of the pairs, and a magnitude.

    Pair i is channels (i, i + n) of n frequencies or, if ``interleaved``,
    (2 i, 2 i + 1); channels from 2 n on are left as they are.  Frequencies are
    kept as the nearest 64-bit fractions of FP64's turn (2^-54 of its value from the
    turn): up to 2^31 radians an angle is off by less than its rounding to FP32."""

    def __init__(self, frequencies, *, interleaved: bool = False, magnitude: float = 1.0,
                 device="cuda"):
        values = torch.as_tensor(frequencies, dtype=torch.float64, device="cpu").flatten().tolist()
        self.dim = 2 * _whole(len(values), "the number of frequencies", 1,
                              kernels.MAX_ROTARY_DIM // 2)
        if not all(map(math.isfinite, values)):
            raise ValueError("frequencies must be finite")
        if not math.isfinite(magnitude):
            raise ValueError("magnitude must be finite")
        self.interleaved, self.magnitude = bool(interleaved), float(magnitude)
        turn = Fraction(2 * math.pi)
        turns = [round(Fraction(f) * 2 ** 64 / turn) % 2 ** 64 for f in values]
        self.turns = torch.tensor([t - 2 ** 64 if t >= 2 ** 63 else t for t in turns],
                                  dtype=torch.int64).to(device)

    def to(self, device) -> "Rotary":
        self.turns = self.turns.to(device)
        return self


_ROTARY_TYPES = tuple(kernels.TYPES)
_MAX_HEADS = 4096


def _check_rotary(plan, q) -> None:
    if type(plan) is not Rotary:
        raise TypeError("plan must be a Rotary")
    if plan.turns.device != q.device:
        raise ValueError("plan and q must be on one device")
    if not plan.dim <= q.shape[-1] <= kernels.MAX_ROTARY_DIM:
        raise ValueError(f"heads must have {plan.dim} to {kernels.MAX_ROTARY_DIM} channels, "
                         f"got {q.shape[-1]}")
    if q.shape[-2] > _MAX_HEADS:
        raise ValueError(f"at most {_MAX_HEADS} heads")


def _first_position(value) -> int:
    return _whole(value, "positions", -2 ** 31, 2 ** 31)


class _ApplyRotary(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, plan, positions, start):
        ctx.plan, ctx.start = plan, start
        ctx.save_for_backward(positions)
        ctx.set_materialize_grads(False)
        q_out, k_out = kernels.rotate(plan, q, k, positions, start, False)
        return q_out if k is None else (q_out, k_out)

    @staticmethod
    def backward(ctx, grad_q, grad_k=None):
        # With a graph of the backward pass asked for, a second one is an error.
        if torch.is_grad_enabled():
            return _rotary_backward_once(ctx, grad_q, grad_k)
        return _rotary_backward(ctx, grad_q, grad_k)


def _rotary_backward(ctx, grad_q, grad_k):
    positions, = ctx.saved_tensors
    if grad_q is None and grad_k is not None:
        grad_k, _ = kernels.rotate(ctx.plan, grad_k, None, positions, ctx.start, True)
    elif grad_q is not None:
        grad_q, grad_k = kernels.rotate(ctx.plan, grad_q, grad_k, positions, ctx.start, True)
    return grad_q, grad_k, None, None, None


_rotary_backward_once = once_differentiable(_rotary_backward)


@torch.compiler.disable
def apply_rotary(plan: Rotary, q: Tensor, k: Tensor | None = None, positions=None):
    """``q`` and ``k``, [batch, token, head, channel] of BF16, FP16 or FP32, turned
    by their positions: ``(q, k)``, or ``q`` alone.  ``positions``: None (0, 1, ..),
    the first token's as an integer up to 2^31 or per sequence as [batch], or each
    token's as [batch, token] (INT32; INT64 is held to INT32's range).  Angles and
    products are FP32, rounded once.  Differentiable in ``q`` and ``k``."""
    _check_tensor(q, "q", 4, _ROTARY_TYPES)
    _check_rotary(plan, q)
    if k is not None:
        _check_like(k, "k", q, 4)
        if k.shape[:2] != q.shape[:2] or k.shape[3] != q.shape[3]:
            raise ValueError("q and k must agree in batch, tokens and channels")
        if k.shape[2] > _MAX_HEADS:
            raise ValueError(f"at most {_MAX_HEADS} heads")
    start = 0
    if isinstance(positions, Tensor):
        positions = _indices(positions, "positions", ((q.shape[0],), tuple(q.shape[:2])), q.device)
    elif positions is not None:
        start, positions = _first_position(positions), None
    if q.numel() == 0 or (k is not None and k.numel() == 0):
        if k is None:
            return q.clone()
        # Of the two, one may have heads.
        return tuple(t.clone() if t.numel() == 0 else
                     apply_rotary(plan, t, positions=start if positions is None else positions)
                     for t in (q, k))
    if _recorded(q, k):
        return _ApplyRotary.apply(q, k, plan, positions, start)
    out = kernels.rotate(plan, q, k, positions, start, False)
    return out[0] if k is None else out


@torch.compiler.disable
def rotary_append(plan: Rotary, q: Tensor, k: Tensor, v: Tensor, k_cache: Tensor, v_cache: Tensor,
                  positions: Tensor) -> Tensor:
    """One new token per sequence, in one launch: returns ``q`` [batch, head,
    channel] turned by ``positions`` [batch], and writes ``k``, turned, and ``v``
    to the caches [batch, capacity, head, channel] there.  A position outside the
    cache is not written.  Not differentiable."""
    _check_tensor(q, "q", 3, _ROTARY_TYPES)
    _check_rotary(plan, q)
    _check_like(k, "k", q, 3)
    _check_like(v, "v", q, 3)
    _check_like(k_cache, "k_cache", q, 4)
    _check_like(v_cache, "v_cache", q, 4)
    batch, kv_heads, dim = k.shape
    if v.shape != k.shape or q.shape[0] != batch or q.shape[2] != dim:
        raise ValueError("q, k and v must agree in batch and channels, k and v in heads")
    if (k_cache.shape != v_cache.shape or k_cache.shape[0] != batch
            or k_cache.shape[2] != kv_heads or k_cache.shape[3] != dim):
        raise ValueError("the caches must be [batch, capacity, head, channel] of k's heads")
    if k_cache.stride(3) != 1 or v_cache.stride(3) != 1:
        raise ValueError("the caches' channels must be adjacent")
    for cache in (k_cache, v_cache):
        if 0 in cache.stride() and any(s == 0 and n > 1
                                       for s, n in zip(cache.stride(), cache.shape)):
            raise ValueError("the caches must not be expanded: tokens would overwrite each other")
    if _recorded(q, k, v, k_cache, v_cache):
        raise ValueError(_NO_GRADIENT)
    if kv_heads > _MAX_HEADS or k_cache.shape[1] > kernels.MAX_TOKENS:
        raise ValueError(f"at most {_MAX_HEADS} heads and {kernels.MAX_TOKENS} tokens")
    positions = _indices(positions, "positions", ((batch,),), q.device)
    if q.numel() == 0 or k_cache.numel() == 0:
        raise ValueError("rotary_append needs a token and a cache")
    q = kernels.rotate_into(plan, q, k, v, k_cache, v_cache, positions)
    # Written: a graph that has saved them must notice.
    torch.autograd.graph.increment_version((k_cache, v_cache))
    return q


# ---- attention

_ATTENTION_TYPES = (torch.bfloat16, torch.float16)


_NO_GRADIENT = ("an input requires a gradient, which this operator does not have: "
                "call it under torch.no_grad()")


def _sight(window, sinks, scale, dim: int) -> tuple:
    window = 0 if window is None else _whole(window, "window", 1, kernels.MAX_TOKENS)
    sinks = _whole(sinks, "sinks", 0, kernels.MAX_TOKENS)
    scale = dim ** -0.5 if scale is None else float(scale)
    # The kernels hold it as FP32: it must not vanish there.
    if not (math.isfinite(scale) and 1e-30 <= scale <= 1e30):
        raise ValueError("scale must be positive and finite")
    return window, sinks, scale


def _check_heads(heads: int, kv_heads: int, dim: int) -> None:
    if heads % kv_heads:
        raise ValueError(f"{heads} query heads are not a multiple of {kv_heads} key heads")
    if dim % 8 or not 8 <= dim <= kernels.MAX_HEAD_DIM:
        raise ValueError(f"heads must have a multiple of 8 channels up to "
                         f"{kernels.MAX_HEAD_DIM}, got {dim}")


class _WindowAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, lengths, window, sinks, scale):
        out, lse = kernels.attention_forward(q, k, v, window, sinks, scale, lengths, True)
        ctx.save_for_backward(q, k, v, out, lse, lengths)
        ctx.sight = window, sinks, scale
        return out

    @staticmethod
    def backward(ctx, grad):
        if torch.is_grad_enabled():
            return _attention_backward_once(ctx, grad)
        return _attention_backward(ctx, grad)


def _attention_backward(ctx, grad):
    q, k, v, out, lse, lengths = ctx.saved_tensors
    return (*kernels.attention_backward(grad, q, k, v, out, lse, *ctx.sight, lengths), None, None,
            None, None)


_attention_backward_once = once_differentiable(_attention_backward)


def check_attention(q, k, v, window, sinks, scale, lengths) -> tuple:
    """:func:`window_attention`'s checks; its ``(window, sinks, scale, lengths)``
    as the kernels take them."""
    _check_tensor(q, "q", 4, _ATTENTION_TYPES)
    _check_like(k, "k", q, 4)
    _check_like(v, "v", q, 4)
    batch, heads, queries, dim = q.shape
    if k.shape != v.shape or k.shape[0] != batch or k.shape[3] != dim:
        raise ValueError("q, k and v must agree in batch and channels, k and v in shape")
    if k.shape[1] == 0 or heads == 0:
        raise ValueError("q and k need at least one head")
    _check_heads(heads, k.shape[1], dim)
    if max(queries, k.shape[2]) > kernels.MAX_TOKENS:
        raise ValueError(f"at most {kernels.MAX_TOKENS} tokens")
    if lengths is not None:
        lengths = _indices(lengths, "lengths", ((batch,),), q.device).contiguous()
    return (*_sight(window, sinks, scale, dim), lengths)


@torch.compiler.disable
def window_attention(q: Tensor, k: Tensor, v: Tensor, *, window: int | None = None, sinks: int = 0,
                     scale: float | None = None, lengths: Tensor | None = None) -> Tensor:
    """Causal attention of [batch, head, token, channel] BF16 or FP16 tensors
    (any strides; token-major storage is read as it is).

    Query i stands at position ``i + keys - queries`` and sees key j where j is
    not later and, with a ``window``, ``position - j < window`` or ``j < sinks``.
    ``lengths`` [batch]: sequence b has that many tokens of the keys', the rest is
    padding that no query sees and whose queries see nothing.  A query that sees
    nothing has output zero and gives no gradient.  ``k`` and ``v`` may have fewer
    heads: query head h reads key head ``h // (heads / key heads)``.  Channels: a
    multiple of 8 up to 128.  ``scale``: positive, channels ** -0.5 if None.

    Scores, softmax and sums are FP32; the softmax weights are rounded to the
    inputs' type for the product with ``v``.  Differentiable in q, k and v; results
    do not depend on timing."""
    window, sinks, scale, lengths = check_attention(q, k, v, window, sinks, scale, lengths)
    if q.numel() == 0 or k.shape[2] == 0:
        # Nothing to compute, or nothing to see: zero whatever q holds, with zero
        # gradients.
        return torch.zeros_like(q) + sum(t[..., :0].sum() for t in (q, k, v))
    if _recorded(q, k, v):
        return _WindowAttention.apply(q, k, v, lengths, window, sinks, scale)
    return kernels.attention_forward(q, k, v, window, sinks, scale, lengths, False)[0]


@torch.compiler.disable
def decode_attention(q: Tensor, k_cache: Tensor, v_cache: Tensor, lengths: Tensor, *,
                     window: int | None = None, sinks: int = 0,
                     scale: float | None = None) -> Tensor:
    """Attention of one query per sequence, ``q`` [batch, head, channel], over
    caches [batch, capacity, head, channel] that hold ``lengths`` [batch] tokens,
    the query's own last: :func:`window_attention` of that token.  A length of 0
    gives zeros; lengths above the capacity count as the capacity.  Of the keys,
    tiles of 32 that hold some that are seen are read; what is not seen has no
    effect, whatever it holds.  Not differentiable."""
    _check_tensor(q, "q", 3, _ATTENTION_TYPES)
    _check_like(k_cache, "k_cache", q, 4)
    _check_like(v_cache, "v_cache", q, 4)
    if _recorded(q, k_cache, v_cache):
        raise ValueError(_NO_GRADIENT)
    batch, heads, dim = q.shape
    if (k_cache.shape != v_cache.shape or k_cache.shape[0] != batch or k_cache.shape[3] != dim):
        raise ValueError("q and the caches must agree in batch and channels, the caches in shape")
    if k_cache.shape[2] == 0 or heads == 0:
        raise ValueError("q and the caches need at least one head")
    _check_heads(heads, k_cache.shape[2], dim)
    if k_cache.shape[1] > kernels.MAX_TOKENS:
        raise ValueError(f"at most {kernels.MAX_TOKENS} tokens")
    lengths = _indices(lengths, "lengths", ((batch,),), q.device).contiguous()
    window, sinks, scale = _sight(window, sinks, scale, dim)
    if q.numel() == 0 or k_cache.shape[1] == 0:
        return torch.zeros_like(q)
    return kernels.attention_decode(q, k_cache, v_cache, window, sinks, scale, lengths)


class KVCache:
    """Keys and values of ``batch`` sequences, [batch, capacity, head, channel],
    and their lengths (INT32, on the device)."""

    def __init__(self, batch: int, capacity: int, kv_heads: int, head_dim: int, *,
                 dtype=torch.bfloat16, device="cuda"):
        batch, capacity = (_whole(n, name, 1, kernels.MAX_TOKENS)
                           for n, name in ((batch, "batch"), (capacity, "capacity")))
        if dtype not in _ATTENTION_TYPES:
            raise TypeError("the cache holds BF16 or FP16")
        kv_heads = _whole(kv_heads, "kv_heads", 1, _MAX_HEADS)
        head_dim = _whole(head_dim, "head_dim", 8, kernels.MAX_HEAD_DIM)
        _check_heads(kv_heads, kv_heads, head_dim)
        shape = (batch, capacity, kv_heads, head_dim)
        self.k = torch.zeros(shape, dtype=dtype, device=device)
        self.v = torch.zeros(shape, dtype=dtype, device=device)
        self.lengths = torch.zeros(batch, dtype=torch.int32, device=device)
        self._most = 0      # no sequence is longer: kept on the host

    @property
    def capacity(self) -> int:
        return self.k.shape[1]

    def reset(self) -> None:
        """Forget all tokens."""
        self.lengths.zero_()
        self._most = 0

    def _check_room(self, tokens: int) -> None:
        if self._most + tokens > self.capacity:
            raise ValueError(f"the cache holds {self.capacity} tokens, {self._most + tokens} asked")

    def _grow(self, tokens: int) -> None:
        self._check_room(tokens)
        self._most += tokens

    def append(self, plan: Rotary, q: Tensor, k: Tensor, v: Tensor) -> Tensor:
        """One new token for every sequence: ``q``, ``k``, ``v`` [batch, head, channel].
        Returns ``q`` turned; ``k`` (turned) and ``v`` are in the cache."""
        self._check_room(1)
        out = rotary_append(plan, q, k, v, self.k, self.v, self.lengths)
        self.lengths += 1
        self._grow(1)
        return out

    def fill(self, plan: Rotary, q: Tensor, k: Tensor, v: Tensor) -> tuple:
        """The prompts of an empty cache, [batch, token, head, channel], all of one
        length: returns ``q`` and ``k`` turned; ``k`` (turned) and ``v`` are in the cache.
        Not differentiable."""
        if self._most:
            raise ValueError("fill() takes an empty cache")
        _check_like(k, "k", self.k, 4)
        _check_like(v, "v", self.k, 4)
        batch, tokens, *heads = k.shape
        if v.shape != k.shape or batch != self.k.shape[0] or tuple(heads) != self.k.shape[2:]:
            raise ValueError("k and v must be [batch, token, head, channel] of the cache's heads")
        if _recorded(q, k, v):
            raise ValueError(_NO_GRADIENT)
        self._check_room(tokens)
        q, k = apply_rotary(plan, q, k)
        self.k[:, :tokens] = k
        self.v[:, :tokens] = v
        self.lengths.fill_(tokens)
        self._grow(tokens)
        return q, k

    def attend(self, q: Tensor, *, window: int | None = None, sinks: int = 0,
               scale: float | None = None) -> Tensor:
        """:func:`decode_attention` of ``q`` over the cache."""
        return decode_attention(q, self.k, self.v, self.lengths, window=window, sinks=sinks,
                                scale=scale)
