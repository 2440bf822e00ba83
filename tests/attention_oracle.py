"""Plain 64-bit forms of the attention path's operators, and how far a kernel's
results may be from them.

The bounds follow the kernels' arithmetic: products and sums in FP32 (2^-24 per
operation, counted generously), the softmax weights and score gradients rounded
to the tensors' type (`unit`: 2^-8 for BF16, 2^-11 for FP16), delta from the
rounded output, one rounding of each result.
"""
from __future__ import annotations

import numpy as np
import torch

UNIT = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
# Half the least step of a type near zero.
LEAST = {torch.bfloat16: 2.0 ** -134, torch.float16: 2.0 ** -25, torch.float32: 2.0 ** -150}
STEP = 2.0 ** -24


def sees(queries, keys, window=None, sinks=0, lengths=None, batch=1):
    """[batch, 1, queries, keys] truth values."""
    position = torch.arange(queries).view(-1, 1) + keys - queries
    key = torch.arange(keys)
    seen = key <= position
    if window is not None:
        seen = seen & ((position - key < window) | (key < sinks))
    seen = seen.expand(batch, 1, queries, keys)
    if lengths is not None:
        length = torch.tensor(lengths).view(-1, 1, 1, 1)
        seen = seen & (key < length) & (position < length)
    return seen


def attention(q, k, v, seen, scale):
    """(out, weights) in 64 bits; rows that see nothing are zero."""
    group = q.shape[1] // k.shape[1]
    k, v = (t.double().repeat_interleave(group, 1) for t in (k, v))
    s = (scale * (q.double() @ k.transpose(-1, -2))).masked_fill(~seen, -float("inf"))
    s = s - s.amax(-1, keepdim=True).clamp(min=-1e300)
    p = s.exp()
    p = p / p.sum(-1, keepdim=True).clamp(min=1e-300)
    return p @ v, p


def attention_with_bounds(q, k, v, seen, scale, grad=None):
    """{name: (exact, bound)} of out and, with `grad`, dq, dk and dv."""
    unit, least = UNIT[q.dtype], LEAST[q.dtype]
    kv_heads, group, dim = k.shape[1], q.shape[1] // k.shape[1], q.shape[3]
    keys = k.shape[2]
    out, p = attention(q, k, v, seen, scale)
    kk, vv = (t.double().repeat_interleave(group, 1) for t in (k, v))
    q, size = q.double(), None
    # A weight's relative error: its score's error, the exponential, the sum.
    size = scale * (q.abs() @ kk.abs().transpose(-1, -2)).amax(-1, keepdim=True)
    weight = 2 * STEP * (keys + (dim + 4) * size + 16)
    bound_out = ((unit + weight) * p) @ vv.abs() + unit * out.abs() + least * (2 + keys)
    result = {"out": (out, bound_out)}
    if grad is None:
        return result
    g = grad.double()
    dp = g @ vv.transpose(-1, -2)
    delta = (g * out).sum(-1, keepdim=True)
    ds = p * (dp - delta)
    error_dp = dim * STEP * (g.abs() @ vv.abs().transpose(-1, -2))
    error_delta = (g.abs() * (bound_out + dim * STEP * out.abs())).sum(-1, keepdim=True)
    error_ds = (p * ((unit + weight + 4 * STEP) * (dp - delta).abs()
                     + (error_dp + error_delta) * (1 + unit + weight)) + least)
    error_ds = error_ds.masked_fill(~seen, 0.0)
    rows = q.shape[2]

    def shared(t):
        return t.unflatten(1, (kv_heads, group)).sum(2)

    dq = scale * (ds @ kk)
    result["dq"] = (dq, scale * ((error_ds + keys * STEP * ds.abs()) @ kk.abs())
                    + unit * dq.abs() + least)
    dk = scale * shared(ds.transpose(-1, -2) @ q)
    result["dk"] = (dk, scale * shared((error_ds + 4 * rows * group * STEP * ds.abs())
                                       .transpose(-1, -2) @ q.abs()) + unit * dk.abs() + least)
    dv = shared(p.transpose(-1, -2) @ g)
    error_p = (unit + weight + 4 * rows * group * STEP) * p + least * seen
    result["dv"] = (dv, shared(error_p.transpose(-1, -2) @ g.abs()) + unit * dv.abs() + least)
    return result


def turned(x, positions, frequencies, interleaved=False, magnitude=1.0, back=False):
    """[batch, token, head, channel] as complex numbers, turned by [batch, token]
    positions, in 64 bits on the host."""
    x = x.detach().cpu().double().clone()
    frequencies = torch.as_tensor(frequencies, dtype=torch.float64)
    n = frequencies.numel()
    angle = positions.cpu().double().unsqueeze(-1) * frequencies
    turn = torch.polar(torch.full_like(angle, magnitude), -angle if back else angle).unsqueeze(2)
    first, second = ((slice(0, 2 * n, 2), slice(1, 2 * n, 2)) if interleaved
                     else (slice(0, n), slice(n, 2 * n)))
    z = torch.complex(x[..., first], x[..., second]) * turn
    x[..., first], x[..., second] = z.real, z.imag
    return x


def turned_bound(x, dtype, exact, frequencies, interleaved=False, magnitude=1.0):
    """One rounding, and FP32 steps on both channels of a pair: the angle (2^-24
    of half a turn), sine and cosine, two products and a sum."""
    n = torch.as_tensor(frequencies).numel()
    x = x.detach().cpu().double().abs()
    if interleaved:
        pair = (x[..., 0:2 * n:2] + x[..., 1:2 * n:2]).repeat_interleave(2, -1)
    else:
        pair = (x[..., :n] + x[..., n:2 * n]).repeat(1, 1, 1, 2)
    bound = torch.zeros_like(x)
    bound[..., :2 * n] = 16 * STEP * abs(magnitude) * pair
    return bound + UNIT[dtype] * exact.abs() + LEAST[dtype]


def philox_words(groups, seed, offset):
    """uint32 [groups, 4]: Philox-4x32-10 at counters (i, offset) under `seed`."""
    c = [np.arange(groups, dtype=np.uint64) & np.uint64(0xFFFFFFFF),
         np.arange(groups, dtype=np.uint64) >> np.uint64(32),
         np.full(groups, offset & 0xFFFFFFFF, dtype=np.uint64),
         np.full(groups, offset >> 32 & 0xFFFFFFFF, dtype=np.uint64)]
    k = [seed & 0xFFFFFFFF, seed >> 32 & 0xFFFFFFFF]
    low, half = np.uint64(0xFFFFFFFF), np.uint64(32)
    for _ in range(10):
        x, y = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        c = [(y >> half) ^ c[1] ^ np.uint64(k[0]), y & low,
             (x >> half) ^ c[3] ^ np.uint64(k[1]), x & low]
        k = [(k[0] + 0x9E3779B9) & 0xFFFFFFFF, (k[1] + 0xBB67AE85) & 0xFFFFFFFF]
    return np.stack(c, 1).astype(np.uint32)


def kept(n, p, seed, offset):
    """The mask of n values."""
    words = philox_words(-(-n // 8), seed, offset)
    halves = np.ascontiguousarray(words.astype("<u4")).view("<u2").reshape(-1)[:n]
    return torch.from_numpy(halves >= round(p * 65536))
