"""Launches of the kernels that are made of matrix products: the cross entropy of a
projection onto a vocabulary (``csrc/cross_entropy.hip``) and Muon's orthogonalisation
(``csrc/orthogonal.hip``).

The callers (``components/losses.py``, ``components/orthogonal.py``,
``components/layers.py``) have checked types and shapes; here tensors get the
strides and alignment that the kernels read, outputs and workspaces are
allocated on the current stream, and the work is shared out.
"""
from __future__ import annotations

from functools import lru_cache
from heapq import heapreplace

import torch
from torch import Tensor

from . import hip
from .attention import TYPES, _check_unrecorded, _launch

MAX_TOKENS = 1 << 22    # LCT_MAX_CROSS_ENTROPY_TOKENS
MAX_VOCAB = 1 << 24     # LCT_MAX_CROSS_ENTROPY_VOCAB
MAX_DIM = 1 << 16       # LCT_MAX_CROSS_ENTROPY_DIM
MAX_LOGITS = 1 << 37    # LCT_MAX_CROSS_ENTROPY_LOGITS

_CUS = 256
_EXACT_TOKENS = 128     # LCT_CROSS_ENTROPY_EXACT_TOKENS
_BIAS_TOKENS = 192      # LCT_CROSS_ENTROPY_BIAS_TOKENS
_PIECE_BYTES = 256 << 20
# Parts of the sum for the gradient of x, of which vocabulary_pieces chooses; 32
# (LCT_MAX_CROSS_ENTROPY_SPLITS) at most.  us of a step with 1 | 2 | 4 | 8 | 16 | 32 parts,
# 50304 x 768: 136 tokens 934 | 519 | 309 | 206 | 157 | 139; 1024: 1109 | 695 | 488 | 391 | 374 |
# 384; 4096: 1750 | 1348 | 1219 | 1268 | 1363 | 1528; 8192: 2449 | 2525 | 2490 | 2643 | 2991 | 3744.
# 32000 x 4096: 512: 1010 | 754 | 655 | 629 | 645 | 704.
_SPLITS = 1, 2, 3, 4, 6, 8, 12, 16, 24, 32

MAX_MATRIX_DIM = 1 << 16    # LCT_MAX_ORTHOGONAL_DIM
MAX_TILES = 1 << 23         # LCT_MAX_ORTHOGONAL_TILES
_NORM_PARTS = 1024          # LCT_ORTHOGONAL_NORM_PARTS
_SPLIT_DEPTH = 2048         # LCT_ORTHOGONAL_SPLIT_DEPTH
_SPLIT_BYTES = 1 << 25      # LCT_ORTHOGONAL_SPLIT_BYTES
_SMALL = 128, 256           # LCT_ORTHOGONAL_SMALL_ROWS, _COLS


def _whole_rows(t: Tensor) -> Tensor:
    """``t``, or a copy, as a matrix whose rows are whole 16-byte pieces at strides and
    an address that the kernels read; zeros where it has to be widened."""
    rows, cols = t.shape
    if cols % 8:
        # Zeros in the last columns alone, where writing the others twice costs more than one
        # more call: us of a call, either | all zeros first: 7 tokens against 53276 x 911 62 |
        # 89, 2 against 37334 x 2250 with gradients 469 | 516, 37 against 307 x 71 202 | 194.
        if rows * cols < 1 << 20:
            out = t.new_zeros(rows, _up8(cols))
        else:
            out = t.new_empty(rows, _up8(cols))
            out[:, cols:] = 0
        out[:, :cols] = t
        return out
    stride = t.stride(0) if rows > 1 else cols
    if (t.stride(1) == 1 and cols <= stride <= MAX_DIM and not stride & 7
            and not t.data_ptr() & 15):
        return t if t.stride(0) == stride else t.as_strided(t.shape, (stride, 1))
    return t.clone(memory_format=torch.contiguous_format)


def _cross_entropy(x: Tensor, weight: Tensor, bias, targets: Tensor, softcap: float,
                   ignore_index: int) -> bytes:
    return hip.CROSS_ENTROPY.pack(
        x.data_ptr(), weight.data_ptr(), 0 if bias is None else bias.data_ptr(),
        targets.data_ptr(), x.stride(0), weight.stride(0), ignore_index, x.shape[0],
        weight.shape[0], x.shape[1], x.dtype == torch.float16, targets.dtype == torch.int64,
        softcap)


def _places(*sizes: int) -> list:
    """Where several working arrays lie in one allocation, each at a multiple of 256 bytes,
    and its size."""
    places, total = [], 0
    for size in sizes:
        places.append(total)
        total += size + 255 & ~255
    places.append(total)
    return places


_FEW_TOKENS = 32        # as many as one tile of the kernel for few tokens has
# Tokens up to which all are multiplied, whether they count or not: finding out and gathering
# costs 6 to 10 us (49 | 38 us with and without of 257 and 256 tokens against 50304 x 768).
_GATHER_TOKENS = 256


def cross_entropy_forward(x: Tensor, weight: Tensor, bias, targets: Tensor, softcap: float,
                          ignore_index: int, reduction: str, keep: bool):
    """``(out, stats)`` of [token, channel] and [vocabulary, channel] matrices, an FP32 bias
    or None and contiguous targets.  ``out``: the losses or, unless the reduction is
    "none", their sum or mean; ``stats`` [2, token], if to ``keep``: the losses and their
    softmax's statistics for :func:`cross_entropy_backward`."""
    _check_unrecorded(x, weight, bias)
    x, weight = _whole_rows(x), _whole_rows(weight)
    tokens, dim = x.shape
    device = x.device
    floats = 8 * tokens * -(-weight.shape[0] // (128 if tokens <= _FEW_TOKENS else 256))
    ints = 1 + 2 * tokens if tokens > _GATHER_TOKENS else 0
    halves = tokens * dim if ints else 0
    at = _places(4 * floats, 4 * ints, 2 * halves, 0 if keep else 8 * tokens)
    memory = torch.empty(at[4], dtype=torch.uint8, device=device)
    base = memory.data_ptr()
    stats = torch.empty((2, tokens), dtype=torch.float32, device=device) if keep else None
    losses = stats.data_ptr() if keep else base + at[3]
    lse, total = losses + 4 * tokens, None
    if reduction != "none":
        out = torch.empty((), dtype=torch.float32, device=device)
        total = out.data_ptr()
    elif keep:
        out = stats[0]
    else:
        out = torch.empty(tokens, dtype=torch.float32, device=device)
        losses = out.data_ptr()
    _launch("lct_cross_entropy_forward", x.get_device(),
            _cross_entropy(x, weight, bias, targets, softcap, ignore_index),
            base + at[1] if ints else None, ints, base + at[2], halves, base, floats, lse, losses,
            total, reduction == "mean")
    return out, stats


def _last_end(lengths, slots: int) -> float:
    """When the last of (how many, how long) workgroups ends that start in this order,
    each as soon as one of the slots is free."""
    free = [0.0] * slots
    for count, length in lengths:
        rounds = max(0, count // slots - 2)
        if rounds:
            # As many for each slot, about: they stay as far apart.
            free = [t + rounds * length for t in free]
        for _ in range(count - rounds * slots):
            heapreplace(free, free[0] + length)
    return max(free)


@lru_cache(maxsize=4096)
def _parts(tokens: int, piece: int, vocab: int, dims: int) -> int:
    """Into how many parts the sum for the gradient of x is divided: those with which a
    piece's products end first, counted in their steps of 32 (as if the weight's gradient
    were needed too)."""
    # The kernel for up to _EXACT_TOKENS takes tiles of 128, two at once per compute unit,
    # and multiplies twice; that for more takes tiles of 256, one at once.
    tile, at_once, twice = (128, 2, 2) if tokens <= _EXACT_TOKENS else (256, 1, 1)
    hidden, weight = dims * -(-tokens // tile), dims * -(-piece // tile)
    # A workgroup's start and end take about as long as 8 steps, reading what earlier pieces
    # left likewise; a value of a part to write and add is 4e-6 of a step.  (Fitted to the
    # times of 13 sizes: what is chosen is within 0.4 % of the best of each.)
    ends = 8 * (2 - piece / max(piece, vocab))
    best = None
    for splits in _SPLITS:
        if splits > max(1, piece // 512):
            break
        time = 4e-6 * splits * tokens * dims * 256 + _last_end(
            ((weight, twice * tokens / 32 + 8),
             (hidden * splits, twice * piece / 32 / splits + ends)),
            at_once * _CUS)
        if best is None or time < best[0]:
            best = time, splits
    return best[1]


def _dz_values(tokens: int) -> int:
    """Values of the logits' gradients per word: whole 16-byte pieces, twice where what
    rounding them leaves is kept."""
    return _up8(tokens) * (2 if tokens <= _EXACT_TOKENS else 1)


def vocabulary_pieces(tokens: int, vocab: int, dim: int) -> tuple:
    """The size of a piece and the parts of its sum for the gradient of x."""
    pieces = -(-vocab * _dz_values(tokens) * 2 // _PIECE_BYTES)
    piece = -(-vocab // (256 * pieces)) * 256
    # (By whole tiles: choosing takes milliseconds.)
    return piece, _parts(-(-tokens // 128) * 128, piece, vocab, -(-dim // 256))


def cross_entropy_backward(grad: Tensor, x: Tensor, weight: Tensor, bias, targets: Tensor,
                           stats: Tensor, softcap: float, ignore_index: int, reduction: str,
                           needed: tuple):
    """``(grad_x, grad_weight, grad_bias)``, None where not ``needed``; the bias's in
    FP32."""
    _check_unrecorded(grad, x, weight, bias)
    dim = x.shape[1]
    x, weight = _whole_rows(x), _whole_rows(weight)
    tokens, width = x.shape
    vocab = weight.shape[0]
    piece, splits = vocabulary_pieces(tokens, vocab, width)
    need_x, need_weight, need_bias = needed
    grad_x = x.new_empty(tokens, width) if need_x else None
    grad_weight = x.new_empty(vocab, width) if need_weight else None
    grad_bias = x.new_empty(vocab, dtype=torch.float32) if need_bias else None
    ints, floats, halves = 1 + 2 * tokens, 1 + 3 * tokens, tokens * width
    dz_size = 0
    if need_x or need_weight:
        dz_size = min(piece, vocab) * _dz_values(tokens)
    hidden_floats = splits * tokens * width if need_x else 0
    bias_floats = 2 * -(-tokens // _BIAS_TOKENS) * vocab if need_bias else 0
    *places, size = _places(4 * ints, 4 * floats, 2 * halves, 2 * dz_size, 4 * hidden_floats,
                            4 * bias_floats)
    memory = torch.empty(size, dtype=torch.uint8, device=x.device)
    base = memory.data_ptr()
    index, values, gathered, dz, hidden, columns = (base + p for p in places)

    def at(t):
        return 0 if t is None else t.data_ptr()

    losses = stats.data_ptr()
    _launch("lct_cross_entropy_backward", x.get_device(),
            _cross_entropy(x, weight, bias, targets, softcap, ignore_index),
            hip.CROSS_ENTROPY_GRADIENTS.pack(
                grad.data_ptr(), losses + 4 * tokens, losses, at(grad_x), at(grad_weight),
                at(grad_bias), index, values, gathered, dz, hidden, columns, ints, floats, halves,
                dz_size, hidden_floats, bias_floats, reduction == "none", reduction == "mean",
                piece, splits))
    if width != dim:
        grad_x, grad_weight = (None if g is None else g[:, :dim].contiguous()
                               for g in (grad_x, grad_weight))
    return grad_x, grad_weight, grad_bias


def _up8(n: int) -> int:
    return -(-n // 8) * 8


def _is_small(rows: int, cols: int) -> bool:
    """Whether one workgroup computes such a matrix (rows <= cols)."""
    return rows <= _SMALL[0] and cols <= _SMALL[1]


def orthogonal_tiles(count: int, rows: int, cols: int) -> int:
    """Workgroups of the largest launch for that many matrices: fewer than MAX_TILES."""
    if _is_small(min(rows, cols), max(rows, cols)):
        return count
    return count * -(-rows // 64) * -(-cols // 64)


def orthogonalize(g: Tensor, steps: int, scale: float, eps: float) -> Tensor:
    """BF16 matrices of [matrix, row, column] ones."""
    _check_unrecorded(g)
    out = torch.empty(g.shape, dtype=torch.bfloat16, device=g.device)
    count, rows, cols = g.shape
    stride, out_stride = g.stride(), out.stride()
    if rows > cols:
        rows, cols = cols, rows
        stride = stride[0], stride[2], stride[1]
        out_stride = out_stride[0], out_stride[2], out_stride[1]
    workspace, size = None, 0
    if not _is_small(rows, cols):
        r, c = _up8(rows), _up8(cols)
        size = (count * (8 * _NORM_PARTS + 6 * r * (c + r))
                + (_SPLIT_BYTES if c >= _SPLIT_DEPTH else 0))
        workspace = torch.empty(size, dtype=torch.uint8, device=g.device)
    _launch("lct_orthogonalize", g.get_device(), hip.ORTHOGONAL.pack(
        g.data_ptr(), out.data_ptr(), *stride, *out_stride, count, rows, cols, steps,
        TYPES[g.dtype], scale, eps), None if workspace is None else workspace.data_ptr(), size)
    return out
