"""The Newton-Schulz iteration of Muon as kernels of its own.

``components/sparse_utils.py``'s ``zeropower_via_newtonschulz5`` (the reference's,
``LCT/components/sparse_utils.py:71-86``) iterates in BF16 on the library's products.
:func:`orthogonalize` computes the same polynomial with the symmetric products by
half and the iterate in 32 bits; ``SparseMuon(fused=True)`` steps with it.
"""
from __future__ import annotations

import math

import torch
from torch import Tensor

from ..kernels import products as kernels
from .attention import _check_tensor, _whole

__all__ = ["orthogonalize"]

_EPS = 1e-7


def check_orthogonalize(G, steps, count: int | None = None) -> int:
    """``steps`` of checked arguments; ``count``: of matrices like ``G``'s, if not its own."""
    if not isinstance(G, Tensor) or G.ndim < 2:
        raise TypeError("G must be a torch.Tensor of at least two dimensions")
    _check_tensor(G, "G", G.ndim, tuple(kernels.TYPES))
    steps = _whole(steps, "steps", 0, 1000)
    rows, cols = G.shape[-2:]
    if max(rows, cols) > kernels.MAX_MATRIX_DIM:
        raise ValueError(f"at most {kernels.MAX_MATRIX_DIM} rows and columns")
    count = math.prod(G.shape[:-2]) if count is None else count
    if kernels.orthogonal_tiles(count, rows, cols) >= kernels.MAX_TILES:
        raise ValueError(f"too many matrices: {count} of {rows} x {cols}")
    return steps


@torch.compiler.disable
@torch.no_grad()
def orthogonalize(G: Tensor, steps: int = 5, *, scale: float = 1.0) -> Tensor:
    """``scale`` times the Newton-Schulz approximation of the polar factor of ``G``, a
    matrix or a batch of them in its last two dimensions, of BF16, FP16 or FP32 and any
    strides; BF16, contiguous, in ``G``'s orientation.

    Each matrix is divided by its Frobenius norm plus 1e-7, then ``steps`` times ``X <- 2 X
    + (-1.5 A + 0.5 A A) X`` with ``A = X X^T`` (of a tall one: transposed).  X is held in 32
    bits (two FP16 numbers), the products' operands are FP16 at fixed powers of two, their
    sums FP32.  Results, their rounding to BF16 (1.7e-3) aside, are off by up to 7e-4
    sqrt(steps) of the exact iteration's norm (2e-4 sqrt(steps) of matrices of a hundred rows
    or more), whatever the norm of ``G``.  In directions in which ``G`` has next to nothing,
    FP32's roundings double with each step, as they do in any FP32 iteration: a matrix of
    rank 1 ends another 2^(steps - 22) of the norm off, 1e-3 after 12 steps but 1e-2 after
    16, so that steps past about 14 are for matrices of full rank.  A call's results are the
    same in every run; in another batch, or at another place of it, a matrix's may differ in
    roundings.  Not differentiable.

    Matrices past 128 x 256 need 6 bytes per value and per value of ``X X^T`` and 8 KiB each
    (with 2048 columns 32 MiB more) while the call runs."""
    steps = check_orthogonalize(G, steps)
    if not abs(scale) <= torch.finfo(torch.float32).max:
        raise ValueError("scale must be finite, in FP32")
    if G.numel() == 0:
        return torch.empty(G.shape, dtype=torch.bfloat16, device=G.device)
    out = kernels.orthogonalize(G.reshape(-1, *G.shape[-2:]), steps, float(scale), _EPS)
    return out.view(G.shape)
