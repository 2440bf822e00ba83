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

import contextlib

import torch
from torch import Tensor

from . import hip

MAX_HEAD_DIM = 128       # LCT_MAX_HEAD_DIM
MAX_ROTARY_DIM = 256     # LCT_MAX_ROTARY_DIM
MAX_TOKENS = 1 << 30

_QUERY_TILE, _KEY_TILE = 128, 64
_DECODE_TILE = 4 * 32    # keys that a workgroup's waves take at a time
_MAX_SPLITS = 64
_CUS = 256

TYPES = {torch.bfloat16: hip.BF16, torch.float16: hip.FP16, torch.float32: hip.FP32}


def on_device(tensor: Tensor):
    """The tensor's device as the current one, for the launch."""
    if tensor.get_device() == torch._C._cuda_getDevice():
        return contextlib.nullcontext()
    return torch.cuda.device(tensor.device)


def _stream(tensor: Tensor) -> int:
    return torch._C._cuda_getCurrentRawStream(tensor.get_device())


def _strides(t: Tensor) -> tuple:
    """Strides of all dimensions but the last; 0 where there is one element."""
    return tuple([0 if n == 1 else s for n, s in zip(t.shape[:-1], t.stride())])


def _readable(t: Tensor) -> Tensor:
    """``t``, or a copy with strides and alignment that the attention kernels
    read: [batch, head, token, channel], 16-byte rows."""
    b, h, n = _strides(t)
    if (t.stride(3) != 1 and t.shape[3] != 1 or t.data_ptr() & 15 or (b | h | n) & 7
            or n >= 1 << 24):
        return t.clone(memory_format=torch.contiguous_format)
    return t


def _btHD(like: Tensor) -> Tensor:
    """A new [batch, head, token, channel] tensor in token-major storage."""
    b, h, t, d = like.shape
    return torch.empty((b, t, h, d), dtype=like.dtype, device=like.device).transpose(1, 2)


def _record(q, k, v, out, lse, lengths, window, sinks, scale) -> bytes:
    batch, heads, queries, dim = q.shape
    return hip.ATTENTION.pack(
        q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(),
        0 if lse is None else lse.data_ptr(), 0 if lengths is None else lengths.data_ptr(),
        *_strides(q), *_strides(k), *_strides(v), *_strides(out), batch, heads, k.shape[1],
        queries, k.shape[2], dim, window, sinks, q.dtype == torch.float16, scale)


def _lse(q: Tensor) -> Tensor:
    """A value per query and head, in whole query tiles."""
    tiles = -(-q.shape[2] // _QUERY_TILE)
    return torch.empty(q.shape[0] * q.shape[1] * tiles * _QUERY_TILE, dtype=torch.float32,
                       device=q.device)


def _seen(keys: int, window: int, sinks: int, rows: int) -> int:
    """The most keys that `rows` adjacent queries see."""
    return keys if window == 0 else min(keys, window + rows - 1 + sinks)


def forward_splits(batch: int, heads: int, queries: int, keys: int, window: int,
                   sinks: int) -> int:
    """Workgroups that share a query tile's keys: as many as fill the compute
    units twice where the tiles alone do not, with 4 key tiles each at least."""
    items = batch * heads * -(-queries // _QUERY_TILE)
    if items > _CUS:
        return 1
    tiles = -(-_seen(keys, window, sinks, min(queries, _QUERY_TILE)) // _KEY_TILE)
    return max(1, min(_MAX_SPLITS, 2 * _CUS // items, tiles // 4))


def attention_forward(q: Tensor, k: Tensor, v: Tensor, window: int, sinks: int, scale: float,
                      lengths, need_lse: bool):
    """``(out, lse)``; ``lse`` is what :func:`attention_backward` needs, or None."""
    q, k, v = _readable(q), _readable(k), _readable(v)
    batch, heads, queries, dim = q.shape
    with on_device(q):
        out = _btHD(q)
        lse = _lse(q) if need_lse else None
        splits = forward_splits(batch, heads, queries, k.shape[2], window, sinks)
        floats = batch * heads * queries * splits * (dim + 2) if splits > 1 else 0
        workspace = torch.empty(floats, dtype=torch.float32, device=q.device) if floats else None
        hip.call("lct_attention_forward",
                 _record(q, k, v, out, lse, lengths, window, sinks, scale), splits,
                 workspace.data_ptr() if floats else None, floats, _stream(q))
    return out, lse


def key_block(dim: int) -> int:
    """Keys of a workgroup of the kernel of dk and dv."""
    return 256 if dim > 64 else 128


def backward_splits(batch: int, heads: int, kv_heads: int, queries: int, keys: int, dim: int,
                    window: int, sinks: int) -> tuple:
    """Workgroups that share the queries of a key block without and with sinks.

    Without: what ends first by the steps (of 64 queries) that the busiest compute
    unit takes, and what the parts' sums cost (the traffic of a part's FP32 sums
    is 0.04 steps of one compute unit, over all of them).  With a window all
    blocks see about as many queries, without one the first sees all and the last
    few.  A block with sinks, which all later queries see, gets parts of an
    eighth of the others' length, which fill what the others leave."""
    per_block = key_block(dim)
    blocks, group = -(-keys // per_block), heads // kv_heads
    slots = _CUS if dim > 64 else 2 * _CUS
    steps = -(-min(queries, keys if window == 0 else window + per_block) // 64) * group
    items = batch * kv_heads * blocks
    best = None
    for splits in range(1, min(_MAX_SPLITS, max(1, steps // 4)) + 1):
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
    part = max(4, -(-steps // splits) // 8)
    return splits, max(1, min(_MAX_SPLITS, -(-(-(-queries // 64) * group) // part)))


def attention_backward(grad: Tensor, q: Tensor, k: Tensor, v: Tensor, out: Tensor, lse: Tensor,
                       window: int, sinks: int, scale: float, lengths):
    """``(dq, dk, dv)``."""
    q, k, v, out, grad = (_readable(t) for t in (q, k, v, out, grad))
    batch, heads, queries, dim = q.shape
    kv_heads, keys = k.shape[1], k.shape[2]
    with on_device(q):
        dq, dk, dv = _btHD(q), _btHD(k), _btHD(v)
        delta = _lse(q)
        splits, sink_splits = backward_splits(batch, heads, kv_heads, queries, keys, dim, window,
                                              sinks)
        per_block = key_block(dim)
        blocks = -(-keys // per_block)
        sink_blocks = -(-min(sinks, keys) // per_block) if window else 0
        parts = sink_blocks * sink_splits + (blocks - sink_blocks) * splits
        floats = (batch * kv_heads * parts * 2 * per_block * dim
                  if splits > 1 or (sink_splits > 1 and sink_blocks) else 0)
        workspace = torch.empty(floats, dtype=torch.float32, device=q.device) if floats else None
        hip.call("lct_attention_backward",
                 _record(q, k, v, out, lse, lengths, window, sinks, scale),
                 hip.ATTENTION_GRADIENTS.pack(
                     grad.data_ptr(), dq.data_ptr(), dk.data_ptr(), dv.data_ptr(),
                     delta.data_ptr(), *_strides(grad), *_strides(dq), *_strides(dk),
                     *_strides(dv)),
                 splits, sink_splits, workspace.data_ptr() if floats else None, floats,
                 _stream(q))
    return dq, dk, dv


def decode_splits(batch: int, heads: int, kv_heads: int, capacity: int, window: int,
                  sinks: int) -> int:
    """Workgroups that share a sequence's keys: as many as fill the compute units
    twice, with one tile per wave each at least."""
    items = batch * kv_heads * -(-(heads // kv_heads) // 16)
    tiles = -(-_seen(capacity, window, sinks, 1) // _DECODE_TILE)
    return max(1, min(_MAX_SPLITS, -(-2 * _CUS // items), tiles))


def attention_decode(q: Tensor, k: Tensor, v: Tensor, window: int, sinks: int, scale: float,
                     lengths) -> Tensor:
    """[batch, heads, channel] of queries of that shape over
    [batch, head, token, channel] caches."""
    q, k, v = _readable(q.unsqueeze(2)), _readable(k), _readable(v)
    batch, heads, _, dim = q.shape
    with on_device(q):
        out = torch.empty((batch, heads, 1, dim), dtype=q.dtype, device=q.device)
        splits = decode_splits(batch, heads, k.shape[1], k.shape[2], window, sinks)
        floats = batch * heads * splits * (dim + 2) if splits > 1 else 0
        workspace = torch.empty(floats, dtype=torch.float32, device=q.device) if floats else None
        hip.call("lct_attention_decode",
                 _record(q, k, v, out, None, lengths, window, sinks, scale), splits,
                 workspace.data_ptr() if floats else None, floats, _stream(q))
    return out.squeeze(2)


def rotate(plan, q: Tensor, k, positions, start: int, inverse: bool, cache=None):
    """The rotated ``(q, k)`` of [batch, token, head, channel] tensors (``k`` may
    be None); with ``cache`` = (v, k_cache, v_cache) ``k`` and ``v`` go there."""
    if q.stride(3) != 1 and q.shape[3] != 1:
        q = q.contiguous()
    if k is not None and k.stride(3) != 1 and k.shape[3] != 1:
        k = k.contiguous()
    batch, tokens, heads, dim = q.shape
    zeros = (0, 0, 0)
    with on_device(q):
        q_out = torch.empty((batch, tokens, heads, dim), dtype=q.dtype, device=q.device)
        v = v_out = k_out = None
        if cache is not None:
            v, k_out, v_out = cache
            if v.stride(3) != 1 and v.shape[3] != 1:
                v = v.contiguous()
        elif k is not None:
            k_out = torch.empty(k.shape, dtype=k.dtype, device=k.device)
        given = [0 if t is None else t.data_ptr() for t in (q, k, v, q_out, k_out, v_out)]
        strides = [s for t in (q, k, v, q_out, k_out, v_out)
                   for s in (zeros if t is None else _strides(t))]
        by_token = positions is not None and positions.ndim == 2
        hip.call("lct_rotate", hip.ROTARY.pack(
            *given, plan.turns.data_ptr(), 0 if positions is None else positions.data_ptr(),
            *strides, 0 if positions is None else positions.stride(0),
            positions.stride(1) if by_token else 0, start, batch, tokens, heads,
            0 if k is None else k.shape[2], dim, plan.dim, plan.interleaved, inverse,
            TYPES[q.dtype], k_out.shape[1] if cache is not None else 0, plan.magnitude),
            _stream(q))
    return q_out, k_out


def dropout(x: Tensor, residual, below: int, seed: int, offset: int, more) -> Tensor:
    """``residual + dropout(x)`` of contiguous, 16-byte aligned tensors."""
    with on_device(x):
        out = torch.empty_like(x)
        hip.call("lct_dropout", x.data_ptr(), None if residual is None else residual.data_ptr(),
                 out.data_ptr(), x.numel(), TYPES[x.dtype], below, seed, offset,
                 None if more is None else more.data_ptr(), _stream(x))
    return out
