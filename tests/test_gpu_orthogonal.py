"""Muon's orthogonalisation on the GPU against the iteration in 64 bits
(``tests/product_oracle.py``)."""
from __future__ import annotations

import pytest
import torch

from gpu_util import require_gpu
from losslessly_compressed_tensors_amd.components.orthogonal import orthogonalize
from losslessly_compressed_tensors_amd.kernels import hip
from product_oracle import (
    polar, polar_floor, polar_off, polar_off_in_empty_directions, polar_rest_floor,
)

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
    bound = (polar_off(steps) * exact.square().sum((-2, -1)).sqrt()
             + abs(scale) * polar_floor(steps, g.shape[-1] * g.shape[-2]))
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


@pytest.mark.parametrize("rows,cols", [(64, 64), (63, 65), (64, 128), (40, 129), (64, 256),
                                       (65, 65), (128, 128), (127, 130), (128, 256), (100, 255),
                                       (129, 129), (128, 257)])
def test_either_side_of_the_small_kernels_sizes(rows, cols):
    for steps in (0, 1, 5, 12):
        for shape in ((3, rows, cols), (3, cols, rows)):
            g = _matrix(shape, "falling").to(BF16)
            _assert_polar(orthogonalize(g.cuda(), steps, scale=-0.5), g, steps, -0.5)


def _views(g):
    """The same matrices in other storages."""
    count, rows, cols = g.shape
    yield g
    yield g.mT.contiguous().mT
    wide = torch.full((count, rows, 2 * cols + 3), 7.0, dtype=g.dtype, device=g.device)
    wide[:, :, 3:cols + 3] = g
    yield wide[:, :, 3:cols + 3]
    steps = torch.full((count, rows, 2 * cols), 7.0, dtype=g.dtype, device=g.device)
    steps[:, :, ::2] = g
    yield steps[:, :, ::2]
    yield g.flip(0).flip(0)
    by_matrix = g.permute(1, 2, 0).contiguous().permute(2, 0, 1)
    yield by_matrix


@pytest.mark.parametrize("shape", [(3, 40, 72), (2, 130, 67), (1, 200, 200)])
@pytest.mark.parametrize("dtype", [BF16, FP32])
def test_strides(shape, dtype):
    g = _matrix(shape).to(dtype).cuda()
    base = orthogonalize(g, 5)
    _assert_polar(base, g, 5)
    for view in _views(g):
        assert torch.equal(orthogonalize(view, 5), base)


def test_wide_and_tall_are_each_others_transposes():
    for shape in ((64, 136), (200, 512), (1000, 1537)):
        g = _matrix(shape).to(BF16).cuda()
        assert torch.equal(orthogonalize(g.mT.contiguous(), 5).mT.contiguous(),
                           orthogonalize(g, 5))


@pytest.mark.parametrize("size", [1e-30, 1e-6, 1.0, 1e30])
def test_any_size(size):
    """eps counts below 1e-6; squares do not overflow."""
    for dtype in (BF16, FP32):
        g = (_matrix((72, 136)) * size).to(dtype)
        _assert_polar(orthogonalize(g.cuda(), 5), g, 5)


def test_nothing_and_zeros():
    assert orthogonalize(torch.zeros(0, 5, 7, device="cuda")).shape == (0, 5, 7)
    assert orthogonalize(torch.zeros(5, 0, device="cuda")).shape == (5, 0)
    out = orthogonalize(torch.zeros(3, 40, 24, device="cuda"), 12)
    assert out.shape == (3, 40, 24) and not out.any()


@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_one_matrix_does_not_reach_another(bad):
    g = _matrix((3, 130, 200)).to(FP32)
    clean = orthogonalize(g.cuda(), 5)
    g[1, 7, 9] = bad
    out = orthogonalize(g.cuda(), 5)
    assert out[1].isnan().any()
    assert torch.equal(out[0], clean[0]) and torch.equal(out[2], clean[2])


# Each tile of the products and one and two steps at a time: by the number of 128 x 128 tiles.
RULES = [(1, 300, 300), (40, 200, 256), (50, 256, 520), (1, 1100, 1100), (90, 300, 400),
         (210, 256, 384), (14, 1024, 1152), (2, 2048, 3200)]


@pytest.mark.parametrize("count,rows,cols", RULES)
def test_every_tile(count, rows, cols):
    g = _matrix((1, rows, cols), "falling").to(BF16).cuda().expand(count, rows, cols).clone()
    signs = torch.where(torch.arange(count, device="cuda") % 2 == 0, 1.0, -1.0).to(BF16)
    g *= signs[:, None, None]
    for steps in (4, 5):
        out = orthogonalize(g, steps)
        exact = polar(g[0].cpu(), steps)
        # Equal matrices give equal results; the negatives' differ from them in roundings (the
        # matrix instructions' are not symmetric about zero).
        for first in (0, 1)[:count]:
            off = float((out[first].cpu().double() * float(signs[first]) - exact).norm()
                        / exact.norm())
            assert off <= polar_off(steps)
            assert torch.equal(out[first::2], out[first:first + 1].expand_as(out[first::2]))


# The symmetric products' last tiles share their depth among workgroups: all 190 by 2, the last
# 32 of 544 by 4.  A matrix's sums then are of an order that its place decides: each result is
# near the exact one, but equal matrices' need not be equal.
@pytest.mark.parametrize("count,rows,cols", [(1, 2432, 2440), (4, 2048, 2056)])
def test_tiles_whose_depth_is_shared(count, rows, cols):
    g = _matrix((1, rows, cols), "falling").to(BF16).cuda().expand(count, rows, cols).clone()
    for steps in (4, 5):
        out = orthogonalize(g, steps)
        assert torch.equal(out, orthogonalize(g, steps))
        exact = polar(g[0].cpu(), steps)
        for got in out.cpu().double():
            assert float((got - exact).norm() / exact.norm()) <= polar_off(steps)


def test_streams_and_replays():
    g = _matrix((4, 200, 136)).to(BF16).cuda()
    eager = orthogonalize(g, 5)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        out = orthogonalize(g, 5)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    assert torch.equal(out, eager)
    static = g.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = orthogonalize(static, 5)
    for seed in (1, 2, 3):
        static.copy_(_matrix((4, 200, 136), seed=seed))
        graph.replay()
        expected = orthogonalize(static, 5)
        torch.cuda.synchronize()
        assert torch.equal(out, expected)


def test_results_do_not_depend_on_the_run():
    g = _matrix((5, 333, 517)).to(BF16).cuda()
    first = orthogonalize(g, 12)
    assert all(torch.equal(first, orthogonalize(g, 12)) for _ in range(3))


def test_refusals():
    g = torch.randn(4, 6, device="cuda")
    for args, error in (((g.double(),), TypeError), ((g.cpu(),), ValueError),
                        ((g.to(torch.complex64),), TypeError), ((g, -1), ValueError),
                        ((g, 2.0), TypeError), ((g, 1001), ValueError)):
        with pytest.raises(error):
            orthogonalize(*args)
    with pytest.raises(ValueError, match="scale"):
        orthogonalize(g, 5, scale=float("nan"))
    with pytest.raises(ValueError, match="at most"):
        orthogonalize(torch.zeros(1, (1 << 16) + 1, device="cuda"))
    for size in (1, 130):
        with pytest.raises(ValueError, match="too many"):
            orthogonalize(torch.zeros(1, 1, 1, device="cuda").expand(1 << 23, size, size))
    with pytest.raises(RuntimeError, match="recorded"):
        torch.jit.trace(lambda a: orthogonalize(a), g)
    # A result has no gradient, whoever asks.
    assert not orthogonalize(g.requires_grad_()).requires_grad


# Lines of the result whose stride the tiles' stores take, or more than they take, past 32 bits
# of bytes within a tile, or backwards: with rows or columns adjacent.
@pytest.mark.parametrize("line", [272, 1 << 16, (1 << 16) + 8, 1 << 26, -272, -(1 << 26)])
@pytest.mark.parametrize("tall", [False, True])
def test_results_of_any_strides(tall, line):
    rows, cols, steps = 136, 264, 3
    g = _matrix((rows, cols)).to(BF16).cuda()
    expected = orthogonalize(g, steps)
    lines, length = (cols, rows) if tall else (rows, cols)
    out = torch.full((lines, abs(line)), 7.0, dtype=BF16, device="cuda")
    first = out.data_ptr() + (2 * (lines - 1) * -line if line < 0 else 0)
    strides = (1, line) if tall else (line, 1)
    workspace = torch.empty(1 << 23, dtype=torch.uint8, device="cuda")
    record = hip.ORTHOGONAL.pack(g.data_ptr(), first, rows * cols, cols, 1, 0, *strides, 1, rows,
                                 cols, steps, hip.BF16, 1.0, 1e-7)
    hip.call("lct_orthogonalize", record, workspace.data_ptr(), workspace.numel(),
             torch.cuda.current_stream().cuda_stream)
    got = out[:, :length].flip(0) if line < 0 else out[:, :length]
    assert torch.equal(got.mT if tall else got, expected)
    for i in range(lines):
        assert not (out[i, length:] != 7).any()


@pytest.mark.parametrize("size", [1e-11, 1e-13, 1e-14, 1e-16])
@pytest.mark.parametrize("rows,cols", [(72, 136), (300, 300), (264, 1000), (2048, 2048)])
def test_norms_far_below_eps(rows, cols, size):
    """X is then small as a whole, and held to its own precision all the same."""
    g = _matrix((rows, cols))
    g *= size / g.norm()
    out = orthogonalize(g.cuda(), 5)
    exact = polar(g, 5)
    off = (out.cpu().double() - exact).norm()
    assert off <= polar_off(5) * exact.norm() + polar_rest_floor(5, rows * cols)


@pytest.mark.parametrize("shape", [(96, 160), (300, 140), (256, 256), (768, 768)])
@pytest.mark.parametrize("steps", [14, 16, 18])
def test_directions_that_a_matrix_does_not_have(steps, shape):
    """FP32's roundings there double with every step."""
    g = _matrix(shape, "rank 1")
    exact = polar(g, steps)
    off = float((orthogonalize(g.cuda(), steps).cpu().double() - exact).norm() / exact.norm())
    assert off <= polar_off(steps) + polar_off_in_empty_directions(steps, min(shape))


@pytest.mark.parametrize("shape", [(96, 160), (160, 96), (300, 300)])
@pytest.mark.parametrize("steps", [30, 101, 300])
def test_many_steps(steps, shape):
    g = _matrix(shape)
    _assert_polar(orthogonalize(g.cuda(), steps), g, steps)
    assert polar_off(300) < 0.03      # (a bound that says something)


def test_scales_that_fp32_does_not_hold_are_refused():
    g = torch.randn(4, 6, device="cuda")
    for scale in (1e39, -1e300, float("inf")):
        with pytest.raises(ValueError, match="scale"):
            orthogonalize(g, 5, scale=scale)
    largest = torch.finfo(FP32).max
    assert not orthogonalize(g, 5, scale=largest).isnan().any()
