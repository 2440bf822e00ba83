"""Muon's orthogonalisation on the GPU against the iteration in 64 bits
(``tests/product_oracle.py``)."""
from __future__ import annotations

import pytest
import torch

from gpu_util import require_gpu
from losslessly_compressed_tensors_amd.components.orthogonal import orthogonalize
from product_oracle import polar, polar_off

pytestmark = pytest.mark.gpu
BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32


@pytest.fixture(autouse=True)
def _gpu():
    require_gpu()


def _matrix(shape, kind="plain", seed=0):
    g = torch.Generator().manual_seed(seed)
    rows, cols = shape[-2:]
    rank = min(rows, cols)
    if kind == "plain":
        return torch.randn(shape, generator=g)
    left = torch.randn(*shape[:-2], rows, rank, generator=g)
    right = torch.randn(*shape[:-2], rank, cols, generator=g)
    if kind == "falling":
        return left / torch.arange(1, rank + 1) @ right
    assert kind == "rank 1"
    return left[..., :1] @ right[..., :1, :]


def _assert_polar(got, g, steps, scale=1.0):
    assert got.dtype == BF16 and got.shape == g.shape and got.is_contiguous()
    exact = polar(g.cpu(), steps, scale)
    off = (got.cpu().double() - exact).square().sum((-2, -1)).sqrt()
    bound = polar_off(steps) * exact.square().sum((-2, -1)).sqrt()
    assert (off <= bound).all(), f"{(off / bound).max():.3g} times the bound"


SIZES = [(1, 1), (1, 7), (9, 1), (8, 8), (5, 13), (64, 64), (33, 129), (130, 66), (127, 128),
         (128, 257), (255, 255), (256, 256), (257, 300), (700, 300), (264, 1000), (513, 520)]


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("rows,cols", SIZES)
def test_sizes(rows, cols, dtype):
    g = _matrix((rows, cols)).to(dtype)
    _assert_polar(orthogonalize(g.cuda(), 5), g, 5)


@pytest.mark.parametrize("steps", [0, 1, 2, 3, 12])
@pytest.mark.parametrize("kind", ["plain", "falling", "rank 1"])
def test_steps_and_spectra(kind, steps):
    for shape in ((96, 160), (300, 140)):
        g = _matrix(shape, kind)
        _assert_polar(orthogonalize(g.cuda(), steps, scale=1.75), g, steps, 1.75)


@pytest.mark.parametrize("shape", [(3, 40, 72), (2, 3, 72, 40), (5, 264, 129), (17, 8, 8)])
def test_batches(shape):
    g = _matrix(shape).to(BF16)
    _assert_polar(orthogonalize(g.cuda(), 5), g, 5)
