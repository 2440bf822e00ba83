"""Launches of the attention path's kernels: rotary positions
(``csrc/rotary.hip``), attention with a sliding window and sinks
(``csrc/attention.hip``, ``csrc/attention_decode.hip``) and dropout
(``csrc/dropout.hip``).

The callers (``components/attention.py``, ``components/dropout.py``,
``components/layers.py``) have checked types and shapes; here tensors get the
strides and alignment that the kernels read, outputs and workspaces are
allocated on the current stream, and the work is shared out.
"""
from __future__ import annotations

from functools import lru_cache

import torch
from torch import Tensor
from torch.autograd import forward_ad

from . import hip

MAX_HEAD_DIM = 128       # LCT_MAX_HEAD_DIM
MAX_ROTARY_DIM = 256     # LCT_MAX_ROTARY_DIM
MAX_TOKENS = 1 << 30

_QUERY_TILE, _KEY_TILE = 128, 64
_DECODE_TILE = 4 * 32    # keys that a workgroup's waves take at a time
_MAX_SPLITS = 64        # LCT_MAX_ATTENTION_SPLITS
_MAX_PARTS = 8          # of dk and dv: FP32 copies of both in the workspace
_PART_GAP = 64          # LCT_ATTENTION_PART_GAP
_CUS = 256

TYPES = {torch.bfloat16: hip.BF16, torch.float16: hip.FP16, torch.float32: hip.FP32}


def _launch(name: str, device: int, *args) -> None:
    """An entry point on ``device``'s current stream."""
    if device == torch._C._cuda_getDevice():
        hip.call(name, *args, torch._C._cuda_getCurrentRawStream(device))
    else:
        with torch.cuda.device(device):
            hip.call(name, *args, torch._C._cuda_getCurrentRawStream(device))


def _check_unrecorded(*tensors) -> None:
    """A launch is no operation of torch's, and has none to fall back to: what records
    or differentiates operations as they run would go on with an unwritten result."""
    if torch._C._get_tracing_state() is not None or torch._C._len_torch_dispatch_stack():
        raise RuntimeError("this operator cannot be recorded: a trace or a dispatch mode is active")
    if forward_ad._current_level >= 0 and torch._C._is_fwd_grad_enabled():
        for t in tensors:
            if t is not None and forward_ad.unpack_dual(t).tangent is not None:
                raise RuntimeError("this operator has no forward-mode derivative")


def _readable(t: Tensor) -> Tensor:
    """``t``, or a copy, of four dimensions with strides and alignment that the
    attention kernels read: rows of 16-byte pieces, tokens in dimension 2."""
    b, h, n, c = t.stride()
    if c == 1 and not (b | h | n) & 7 and n < 1 << 24 and not t.data_ptr() & 15:
        return t
    # Dimensions of one element have any stride: only 0 is sure to be in range.
    size = t.shape
    b, h, n = b * (size[0] > 1), h * (size[1] > 1), n * (size[2] > 1)
    if (c == 1 or size[3] == 1) and not (b | h | n) & 7 and n < 1 << 24 and not t.data_ptr() & 15:
        return t.as_strided(size, (b, h, n, 1))
    return t.clone(memory_format=torch.contiguous_format)


def _cache(t: Tensor) -> tuple:
    """A [batch, token, head, channel] cache as :func:`_readable` would have it, and
    its strides of batch, head and token."""
    b, n, h, c = t.stride()
    if c == 1 and not (b | h | n) & 7 and n < 1 << 24 and not t.data_ptr() & 15:
        return t, (b, h, n)
    t = _readable(t.transpose(1, 2)).transpose(1, 2)
    b, n, h, _ = t.stride()
    return t, (b, h, n)


def _token_major(like: Tensor) -> Tensor:
    """A new [batch, head, token, channel] tensor in token-major storage."""
    b, h, t, d = like.shape
    return like.new_empty_strided((b, h, t, d), (t * h * d, d, h * d, 1))


def _record(q, k, v, out, lse, lengths, window, sinks, scale) -> bytes:
    batch, heads, queries, dim = q.shape
    _, kv_heads, keys, _ = k.shape
    return hip.ATTENTION.pack(
        q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(),
        0 if lse is None else lse.data_ptr(), 0 if lengths is None else lengths.data_ptr(),
        *q.stride()[:3], *k.stride()[:3], *v.stride()[:3], *out.stride()[:3], batch, heads,
        kv_heads, queries, keys, dim, window, sinks, q.dtype == torch.float16, scale)


def _lse(q: Tensor) -> Tensor:
    """A value per query and head, in whole query tiles."""
    tiles = -(-q.shape[2] // _QUERY_TILE)
    return q.new_empty(q.shape[0] * q.shape[1] * tiles * _QUERY_TILE, dtype=torch.float32)


def _workspace(q: Tensor, floats: int):
    """FP32 working memory and its address, None for none."""
    if not floats:
        return None, None
    workspace = q.new_empty(floats, dtype=torch.float32)
    return workspace, workspace.data_ptr()


def _seen(keys: int, window: int, sinks: int, rows: int) -> int:
    """The most keys that `rows` adjacent queries see."""
    return keys if window == 0 else min(keys, window + rows - 1 + sinks)


@lru_cache(maxsize=1024)
def forward_splits(batch: int, heads: int, queries: int, keys: int, window: int,
                   sinks: int) -> int:
    """Workgroups that share a query tile's keys: as many as fill the compute
    units twice where there is no tile for each, with 4 key tiles each at least.
    us in one part | two, of a few queries after 16384 keys: 32 tiles of heads of 128
    282 | 153 (84 in four), 256 338 | 288; above the line 300 388 | 400, 384 423 | 426,
    512 491 | 536; of heads of 64 300 278 | 244, 512 314 | 352, 640 407 | 427; 300 of 128
    after 4096 keys 101 | 128."""
    items = batch * heads * -(-queries // _QUERY_TILE)
    if items > _CUS:
        return 1
    tiles = -(-_seen(keys, window, sinks, min(queries, _QUERY_TILE)) // _KEY_TILE)
    return max(1, min(_MAX_SPLITS, 2 * _CUS // items, tiles // 4))


def attention_forward(q: Tensor, k: Tensor, v: Tensor, window: int, sinks: int, scale: float,
                      lengths, need_lse: bool):
    """``(out, lse)``; ``lse`` is what :func:`attention_backward` needs, or None."""
    _check_unrecorded(q, k, v)
    q, k, v = _readable(q), _readable(k), _readable(v)
    batch, heads, queries, dim = q.shape
    out = _token_major(q)
    lse = _lse(q) if need_lse else None
    splits = forward_splits(batch, heads, queries, k.shape[2], window, sinks)
    floats = batch * heads * queries * splits * (dim + 2) if splits > 1 else 0
    workspace, address = _workspace(q, floats)
    _launch("lct_attention_forward", q.get_device(),
            _record(q, k, v, out, lse, lengths, window, sinks, scale), splits, address, floats)
    return out, lse


def key_block(dim: int) -> int:
    """Keys of a workgroup of the kernel of dk and dv."""
    return 256 if dim > 64 else 128


@lru_cache(maxsize=1024)
def backward_splits(batch: int, heads: int, kv_heads: int, queries: int, keys: int, dim: int,
                    window: int, sinks: int) -> tuple:
    """Workgroups that share the queries of a key block without and with sinks.

    Without: what ends first by the steps (of 64 queries) that the busiest compute
    unit takes, and what the parts' sums cost (the traffic of a part's FP32 sums
    is 0.04 steps of one compute unit, over all of them).  With a window all
    blocks see about as many queries, without one the first sees all and the last
    few.  A block with sinks, which all later queries see, gets parts of a
    sixteenth of the others' length, which fill what the others leave."""
    per_block = key_block(dim)
    blocks, group = -(-keys // per_block), heads // kv_heads
    slots = _CUS if dim > 64 else 3 * _CUS
    steps = -(-min(queries, keys if window == 0 else window + per_block) // 64) * group
    items = batch * kv_heads * blocks
    best = None
    for splits in range(1, min(_MAX_PARTS, max(1, steps // 4)) + 1):
        part = -(-steps // splits)
        if window == 0:
            time = items * steps / 2 / slots + part
        else:
            time = -(-items * splits // slots) * part
        time += 0.04 * items * splits / slots * (splits > 1) * _CUS
        if best is None or time < best[0]:
            best = time, splits
    splits = best[1]
    if window == 0 or sinks == 0:
        return splits, 1
    part = max(4, -(-steps // splits) // 16)
    return splits, max(1, min(_MAX_SPLITS, -(-(-(-queries // 64) * group) // part)))


def backward_workspace(batch: int, kv_heads: int, keys: int, dim: int, window: int, sinks: int,
                       splits: int, sink_splits: int) -> int:
    """Floats of the parts of dk and dv: of the key blocks that have several."""
    per_block = key_block(dim)
    sink_blocks = -(-min(sinks, keys) // per_block) if window else 0
    parts = sink_blocks * sink_splits if sink_splits > 1 else 0
    if splits > 1:
        parts += (-(-keys // per_block) - sink_blocks) * splits
    return batch * kv_heads * parts * (2 * per_block * dim + _PART_GAP)


def attention_backward(grad: Tensor, q: Tensor, k: Tensor, v: Tensor, out: Tensor, lse: Tensor,
                       window: int, sinks: int, scale: float, lengths):
    """``(dq, dk, dv)``."""
    _check_unrecorded(grad, q, k, v)
    q, k, v, out, grad = (_readable(t) for t in (q, k, v, out, grad))
    batch, heads, queries, dim = q.shape
    kv_heads, keys = k.shape[1], k.shape[2]
    dq, dk, dv = _token_major(q), _token_major(k), _token_major(v)
    delta = _lse(q)
    splits, sink_splits = backward_splits(batch, heads, kv_heads, queries, keys, dim, window,
                                          sinks)
    floats = backward_workspace(batch, kv_heads, keys, dim, window, sinks, splits, sink_splits)
    workspace, address = _workspace(q, floats)
    _launch("lct_attention_backward", q.get_device(),
            _record(q, k, v, out, lse, lengths, window, sinks, scale),
            hip.ATTENTION_GRADIENTS.pack(
                grad.data_ptr(), dq.data_ptr(), dk.data_ptr(), dv.data_ptr(), delta.data_ptr(),
                *grad.stride()[:3], *dq.stride()[:3], *dk.stride()[:3], *dv.stride()[:3]),
            splits, sink_splits, address, floats)
    return dq, dk, dv


@lru_cache(maxsize=1024)
def decode_splits(batch: int, heads: int, kv_heads: int, capacity: int, window: int,
                  sinks: int) -> int:
    """Workgroups that share a sequence's keys.  Up to 1024 keys one is as fast as
    several with the launch that joins their parts (us at 12 heads: 5.1 | 7.1 at
    257 keys, 7.6 | 7.4 at 1024, two and four parts); above, three workgroups per
    compute unit (8 heads of 8192 keys: 74 in one part, 21 in 6, 13.8 in 24, 16 in
    48; 128 of 4096: 75, 40 in 6, 44 in 8, 60 in 32), with 256 keys each at least,
    and of long caches one part per 24 tiles, if more, up to 64, so that sequences of
    unequal length even out (32 heads of up to 131072: 311 in 16 parts, 278 to 283 in
    24, 275 to 278 in the 42 that they get, 268 to 275 in 64)."""
    items = batch * kv_heads * -(-(heads // kv_heads) // 16)
    tiles = -(-_seen(capacity, window, sinks, 1) // _DECODE_TILE)
    if tiles <= 8:
        return 1
    return max(1, min(_MAX_SPLITS, tiles // 2, max(3 * _CUS // items, tiles // 24)))


def attention_decode(q: Tensor, k_cache: Tensor, v_cache: Tensor, window: int, sinks: int,
                     scale: float, lengths) -> Tensor:
    """[batch, head, channel] of queries of that shape over [batch, token, head,
    channel] caches."""
    _check_unrecorded(q, k_cache, v_cache)
    qb, qh, qc = q.stride()
    if qc != 1 or (qb | qh) & 7 or q.data_ptr() & 15:
        q = q.clone(memory_format=torch.contiguous_format)
        qb, qh, _ = q.stride()
    k_cache, k_stride = _cache(k_cache)
    v_cache, v_stride = _cache(v_cache)
    batch, heads, dim = q.shape
    _, capacity, kv_heads, _ = k_cache.shape
    out = torch.empty_like(q, memory_format=torch.contiguous_format)
    splits = decode_splits(batch, heads, kv_heads, capacity, window, sinks)
    floats = batch * heads * splits * (dim + 2) if splits > 1 else 0
    workspace, address = _workspace(q, floats)
    _launch("lct_attention_decode", q.get_device(), hip.ATTENTION.pack(
        q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), out.data_ptr(), 0,
        0 if lengths is None else lengths.data_ptr(), qb, qh, 0, *k_stride, *v_stride, heads * dim,
        dim, 0, batch, heads, kv_heads, 1, capacity, dim, window, sinks, q.dtype == torch.float16,
        scale), splits, address, floats)
    return out


_NO_STRIDES = (0, 0, 0)


def rotate(plan, q: Tensor, k, positions, start: int, inverse: bool):
    """The rotated ``(q, k)`` of [batch, token, head, channel] tensors; ``k`` may be
    None."""
    _check_unrecorded(q, k)
    if q.stride(3) != 1:
        q = q.contiguous()
    batch, tokens, heads, dim = q.shape
    q_out = torch.empty_like(q, memory_format=torch.contiguous_format)
    if k is None:
        k_out, k_in_at, k_out_at, kv_heads = None, 0, 0, 0
        k_in_stride = k_out_stride = _NO_STRIDES
    else:
        if k.stride(3) != 1:
            k = k.contiguous()
        k_out = torch.empty_like(k, memory_format=torch.contiguous_format)
        k_in_at, k_out_at, kv_heads = k.data_ptr(), k_out.data_ptr(), k.shape[2]
        k_in_stride, k_out_stride = k.stride()[:3], k_out.stride()[:3]
    at = b = t = 0
    if positions is not None:
        if positions.ndim == 2 and positions.stride(1) == 0:
            # A stride of 0 would mean that the sequence's tokens follow each other.
            positions = positions.contiguous()
        at, b = positions.data_ptr(), positions.stride(0)
        t = positions.stride(1) if positions.ndim == 2 else 0
    _launch("lct_rotate", q.get_device(), hip.ROTARY.pack(
        q.data_ptr(), k_in_at, 0, q_out.data_ptr(), k_out_at, 0, plan.turns.data_ptr(), at,
        *q.stride()[:3], *k_in_stride, 0, 0, 0, *q_out.stride()[:3], *k_out_stride, 0, 0, 0, b, t,
        start, batch, tokens, heads, kv_heads, dim, plan.dim, plan.interleaved, inverse,
        TYPES[q.dtype], 0, plan.magnitude))
    return q_out, k_out


def rotate_into(plan, q: Tensor, k: Tensor, v: Tensor, k_cache: Tensor, v_cache: Tensor,
                positions: Tensor) -> Tensor:
    """The rotated ``q`` [batch, head, channel]; ``k``, rotated, and ``v`` go to the
    [batch, token, head, channel] caches at ``positions``."""
    _check_unrecorded(q, k, v, k_cache, v_cache)
    q, k, v = (t if t.stride(2) == 1 else t.contiguous() for t in (q, k, v))
    batch, heads, dim = q.shape
    out = torch.empty_like(q, memory_format=torch.contiguous_format)
    (qb, qh, _), (kb, kh, _), (vb, vh, _) = q.stride(), k.stride(), v.stride()
    _launch("lct_rotate", q.get_device(), hip.ROTARY.pack(
        q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), k_cache.data_ptr(),
        v_cache.data_ptr(), plan.turns.data_ptr(), positions.data_ptr(), qb, 0, qh, kb, 0, kh, vb,
        0, vh, heads * dim, 0, dim, *k_cache.stride()[:3], *v_cache.stride()[:3],
        positions.stride(0), 0, 0, batch, 1, heads, k.shape[1], dim, plan.dim, plan.interleaved,
        False, TYPES[q.dtype], k_cache.shape[1], plan.magnitude))
    return out


def dropout(x: Tensor, residual, below: int, seed: int, offset: int, more) -> Tensor:
    """``residual + dropout(x)`` of contiguous, 16-byte aligned tensors."""
    _check_unrecorded(x, residual)
    out = torch.empty_like(x)
    _launch("lct_dropout", x.get_device(), x.data_ptr(),
            None if residual is None else residual.data_ptr(), out.data_ptr(), x.numel(),
            TYPES[x.dtype], below, seed, offset, None if more is None else more.data_ptr())
    return out
