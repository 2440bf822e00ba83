"""What the product operators refuse, and how their work is shared out (CPU)."""
from __future__ import annotations

import ctypes

import pytest
import torch

from conftest import ROOT  # noqa: F401
from losslessly_compressed_tensors_amd.components.losses import (
    check_cross_entropy, linear_cross_entropy,
)
from losslessly_compressed_tensors_amd.components.orthogonal import orthogonalize
from losslessly_compressed_tensors_amd.components.sparse_utils import SparseMuon
from losslessly_compressed_tensors_amd.kernels import hip, products
from product_oracle import CrossEntropy, polar

E_NULL, E_SIZE, E_ARG = -1, -3, -4


@pytest.fixture(scope="module")
def lib():
    if not hip.LIBRARY_PATH.exists():
        pytest.skip("liblct_hip.so not built (python -m losslessly_compressed_tensors_amd.build)")
    return hip.load_library()


# ---- the oracle itself


def test_oracle_gradients_are_those_of_differences():
    g = torch.Generator().manual_seed(0)
    x = torch.randn(5, 3, generator=g, dtype=torch.float64)
    weight = torch.randn(7, 3, generator=g, dtype=torch.float64).float()
    bias = torch.randn(7, generator=g, dtype=torch.float64)
    targets = torch.tensor([0, 6, -100, 3, 3])
    for softcap in (None, 2.0):
        for reduction in ("mean", "sum"):
            def total(x, w, b):
                return CrossEntropy(x, w, targets, b, softcap, reduction=reduction).total
            exact = CrossEntropy(x, weight, targets, bias, softcap, reduction=reduction)
            weight64 = weight.double()
            h = 1e-5
            for values, grad, at in ((x, exact.grad_x, 0), (weight64, exact.grad_weight, 1),
                                     (bias, exact.grad_bias, 2)):
                for i in range(values.numel()):
                    ends = []
                    for sign in (1, -1):
                        moved = [x, weight64, bias]
                        moved[at] = values.clone()
                        moved[at].view(-1)[i] += sign * h
                        moved[1] = _Double(moved[1])
                        ends.append(total(moved[0], moved[1], moved[2]))
                    slope = float((ends[0] - ends[1]) / (2 * h))
                    # h^2 of a third derivative below 10, and rounding over h.
                    assert abs(slope - float(grad.reshape(-1)[i])) < 1e-8


class _Double:
    """A weight in 64 bits whose type, for the bounds alone, is another's."""

    def __init__(self, t):
        self.t, self.dtype, self.shape = t, torch.bfloat16, t.shape

    def double(self):
        return self.t


def test_oracle_polar_of_an_orthogonal_matrix_is_itself():
    q, _ = torch.linalg.qr(torch.randn(6, 6, dtype=torch.float64,
                                       generator=torch.Generator().manual_seed(1)))
    # Singular values 6^-1/2 after the division by the norm, then towards 1.
    assert (polar(q, 30) - q).abs().max() < 1e-6


# ---- refusals


class _FakeGpu(torch.Tensor):
    pass


def _args(**changes):
    args = dict(x=torch.zeros(3, 8, dtype=torch.bfloat16),
                weight=torch.zeros(5, 8, dtype=torch.bfloat16),
                targets=torch.zeros(3, dtype=torch.int64), bias=None, softcap=None,
                ignore_index=-100, reduction="mean")
    args.update(changes)
    return args


def test_host_tensors_and_other_kinds_are_refused():
    with pytest.raises(ValueError, match="x must be a GPU tensor"):
        check_cross_entropy(**_args())
    with pytest.raises(TypeError, match="at least one dimension"):
        linear_cross_entropy(3.0, torch.zeros(5, 8), torch.zeros(3))
    with pytest.raises(TypeError, match="at least one dimension"):
        linear_cross_entropy(torch.zeros((), dtype=torch.bfloat16), torch.zeros(5, 8),
                             torch.zeros(()))
    with pytest.raises(TypeError, match="plain"):
        check_cross_entropy(**_args(x=torch.zeros(3, 8).as_subclass(_FakeGpu)))
    with pytest.raises(ValueError, match="G must be a GPU tensor"):
        orthogonalize(torch.zeros(4, 4))
    for bad in (3, torch.zeros(4)):
        with pytest.raises(TypeError, match="at least two dimensions"):
            orthogonalize(bad)


def _cross_entropy(x=1 << 20, weight=1 << 20, bias=0, targets=1 << 20, x_stride=8,
                   weight_stride=8, ignore_index=-100, tokens=3, vocab=5, dim=8, fp16=0,
                   targets_64=1, softcap=0.0):
    return hip.CROSS_ENTROPY.pack(x, weight, bias, targets, x_stride, weight_stride, ignore_index,
                                  tokens, vocab, dim, fp16, targets_64, softcap)


@pytest.mark.parametrize("changes,code", [
    (dict(x=0), E_NULL), (dict(weight=0), E_NULL), (dict(targets=0), E_NULL),
    (dict(tokens=0), E_SIZE), (dict(tokens=(1 << 22) + 1), E_SIZE),
    (dict(tokens=1 << 22, vocab=(1 << 15) + 1), E_SIZE), (dict(vocab=0), E_SIZE),
    (dict(vocab=(1 << 24) + 1), E_SIZE), (dict(dim=0), E_SIZE), (dict(dim=12), E_SIZE),
    (dict(dim=(1 << 16) + 8), E_SIZE), (dict(x_stride=0), E_ARG), (dict(x_stride=12), E_ARG),
    (dict(weight_stride=0), E_ARG), (dict(weight_stride=(1 << 16) + 8), E_ARG),
    (dict(x=(1 << 20) + 8), E_ARG), (dict(weight=(1 << 20) + 2), E_ARG),
    (dict(bias=(1 << 20) + 2), E_ARG), (dict(targets=(1 << 20) + 4), E_ARG),
    (dict(softcap=-1.0), E_ARG), (dict(softcap=float("nan")), E_ARG),
    (dict(softcap=1e20), E_ARG),
])
def test_entry_points_refuse_bad_records_before_a_launch(lib, changes, code):
    record = _cross_entropy(**changes)
    at = 1 << 20     # never dereferenced
    big = 1 << 40
    assert lib.lct_cross_entropy_forward(record, None, 0, None, 0, at, big, at, at, None, 0,
                                         None) == code
    assert lib.lct_cross_entropy_backward(record, _gradients(), None) == code


def _gradients(grad=1 << 20, lse=1 << 20, losses=1 << 20, grad_x=1 << 20, grad_weight=1 << 20,
               grad_bias=0, index=1 << 20, values=1 << 20, gathered=1 << 20, dz=1 << 20,
               hidden=1 << 20, columns=0, index_size=1 << 40, value_floats=1 << 40,
               gathered_size=1 << 40, dz_size=1 << 40, hidden_floats=1 << 40,
               bias_floats=1 << 40, per_token=0, mean=0, piece=256, splits=1):
    return hip.CROSS_ENTROPY_GRADIENTS.pack(
        grad, lse, losses, grad_x, grad_weight, grad_bias, index, values, gathered, dz, hidden,
        columns, index_size, value_floats, gathered_size, dz_size, hidden_floats, bias_floats,
        per_token, mean, piece, splits)


@pytest.mark.parametrize("changes,code", [
    (dict(grad=0), E_NULL), (dict(lse=0), E_NULL), (dict(losses=0), E_NULL),
    (dict(index=0), E_NULL), (dict(values=0), E_NULL), (dict(gathered=0), E_NULL),
    (dict(dz=0), E_NULL), (dict(hidden=0), E_NULL), (dict(grad_bias=1 << 20), E_NULL),
    (dict(piece=0), E_SIZE), (dict(piece=100), E_SIZE), (dict(splits=0), E_SIZE),
    (dict(splits=33), E_SIZE), (dict(index_size=6), E_SIZE), (dict(value_floats=9), E_SIZE),
    (dict(gathered_size=23), E_SIZE), (dict(dz_size=79), E_SIZE), (dict(hidden_floats=23), E_SIZE),
    (dict(gathered=(1 << 20) + 8), E_ARG), (dict(dz=(1 << 20) + 8), E_ARG),
    (dict(grad_x=(1 << 20) + 8), E_ARG), (dict(grad_weight=(1 << 20) + 2), E_ARG),
])
def test_backward_refuses_small_workspaces_before_a_launch(lib, changes, code):
    assert lib.lct_cross_entropy_backward(_cross_entropy(), _gradients(**changes), None) == code


def test_launches_of_too_many_workgroups_are_refused(lib):
    # 256 tiles of channels by 32768 of tokens, and one of the vocabulary.
    record = _cross_entropy(tokens=1 << 22, dim=1 << 16, x_stride=1 << 16, weight_stride=1 << 16)
    assert lib.lct_cross_entropy_backward(record, _gradients(), None) == E_SIZE


def test_tiles_of_an_orthogonalisation():
    assert products.orthogonal_tiles(7, 256, 128) == 7
    assert products.orthogonal_tiles(7, 129, 129) == 7 * 9
    assert products.orthogonal_tiles(1, 257, 1) == 5


def test_forward_refuses_small_workspaces_before_a_launch(lib):
    at = 1 << 20

    def call(index=at, index_size=1 << 30, gathered=at, gathered_size=1 << 30, floats=1 << 30,
             parts=at):
        return lib.lct_cross_entropy_forward(_cross_entropy(), index, index_size, gathered,
                                             gathered_size, parts, floats, at, at, None, 0, None)

    assert call(parts=None) == E_NULL
    assert call(gathered=None) == E_NULL
    assert call(floats=8 * 3 - 1) == E_SIZE
    assert call(parts=at + 4) == E_SIZE
    assert call(index_size=6) == E_SIZE
    assert call(gathered_size=23) == E_SIZE
    assert call(gathered=at + 8) == E_SIZE


@pytest.mark.parametrize("changes,code", [
    (dict(input=0), E_NULL), (dict(out=0), E_NULL), (dict(count=0), E_SIZE),
    (dict(rows=0), E_SIZE), (dict(rows=137), E_SIZE), (dict(cols=(1 << 16) + 1), E_SIZE),
    (dict(steps=-1), E_SIZE), (dict(type=3), E_ARG), (dict(type=-1), E_ARG),
    (dict(count=1 << 23), E_SIZE), (dict(count=1 << 23, rows=8, cols=8), E_SIZE),
    (dict(size=8 * 1024 + 12 * 136 * 136 - 1), E_SIZE),
    (dict(cols=2048, size=8 * 1024 + 6 * 136 * (2048 + 136) + (1 << 25) - 1), E_SIZE),
    (dict(workspace=(1 << 20) + 8), E_ARG), (dict(workspace=None), E_NULL),
])
def test_orthogonalize_entry_point_refuses_before_a_launch(lib, changes, code):
    values = dict(input=1 << 20, out=1 << 20, count=1, rows=136, cols=136, steps=1, type=0,
                  workspace=1 << 20, size=1 << 40)
    values.update(changes)
    record = hip.ORTHOGONAL.pack(values["input"], values["out"], 136 * 136, 136, 1, 136 * 136, 136, 1,
                                 values["count"], values["rows"], values["cols"], values["steps"],
                                 values["type"], 1.0, 1e-7)
    assert lib.lct_orthogonalize(record, values["workspace"], values["size"], None) == code


def test_records_have_the_headers_sizes():
    # Pointers and 64-bit values, then 32-bit ones, padded to 8 bytes.
    assert hip.CROSS_ENTROPY.size == 4 * 8 + 3 * 8 + 6 * 4
    assert hip.CROSS_ENTROPY_GRADIENTS.size == 12 * 8 + 6 * 8 + 4 * 4
    assert hip.ORTHOGONAL.size == 2 * 8 + 6 * 8 + 7 * 4 + 4
    assert ctypes.sizeof(ctypes.c_void_p) == 8


# ---- shares of the work


@pytest.mark.parametrize("tokens", [1, 37, 1013, 8192, 16384, 1 << 20, 1 << 22])
@pytest.mark.parametrize("vocab", [1, 307, 50304, 100352, 1 << 24])
@pytest.mark.parametrize("dim", [8, 768, 4096])
def test_pieces_cover_the_vocabulary_within_their_memory(tokens, vocab, dim):
    piece, splits = products.vocabulary_pieces(tokens, vocab, dim)
    assert piece % 256 == 0 and piece > 0 and 1 <= splits <= 32
    # One tile's width is the least.
    assert 2 * tokens * (piece - 256) <= products._PIECE_BYTES
    assert piece - 256 < vocab or piece == 256


def test_last_end_is_a_list_schedules():
    assert products._last_end(((1, 5.0),), 512) == 5.0
    assert products._last_end(((512, 5.0),), 512) == 5.0
    assert products._last_end(((513, 5.0),), 512) == 10.0
    # 3 slots' worth of long ones, the short ones in the others.
    assert products._last_end(((3, 8.0), (2 * (256 - 3), 4.0)), 256) == 8.0


def test_workspace_arrays_lie_apart_and_aligned():
    assert products._places(1, 0, 300, 256) == [0, 256, 256, 768, 1024]


def test_the_packages_paths_are_the_modules():
    import LCT.components.losses
    import LCT.components.orthogonal
    assert LCT.components.losses.linear_cross_entropy is linear_cross_entropy
    assert LCT.components.orthogonal.orthogonalize is orthogonalize


def test_muon_takes_the_option():
    p = torch.nn.Parameter(torch.zeros(4, 4))
    assert SparseMuon([p], compressed=False).fused is False
    assert SparseMuon([p], compressed=False, fused=True).fused is True


@pytest.mark.parametrize("tokens", [1, 8, 37, 128, 129, 4096])
@pytest.mark.parametrize("vocab", [50304, (1 << 20) + 7, 1 << 24])
def test_both_numbers_of_a_piece_are_within_its_memory(tokens, vocab):
    """Of up to 128 tokens the logits' gradients are held in two numbers, each token's in whole
    pieces of eight."""
    piece, _ = products.vocabulary_pieces(tokens, vocab, 64)
    numbers = 2 if tokens <= 128 else 1
    assert 2 * numbers * -(-tokens // 8) * 8 * (piece - 256) <= 256 << 20


def test_the_biases_parts_are_a_tile_of_tokens_each(lib):
    """Two of 192 tokens and a word: no fewer, and no more are asked for."""
    record = _cross_entropy(tokens=1000, bias=1 << 20)
    for floats, hidden, code in ((2 * 6 * 5 - 1, 1 << 40, E_SIZE), (2 * 6 * 5, 1 << 40, E_ARG)):
        # (An odd address, which is looked at behind the sizes.)
        gradients = _gradients(grad_bias=1 << 20, columns=1 << 20, bias_floats=floats,
                               hidden_floats=hidden, dz=(1 << 20) + 8)
        assert lib.lct_cross_entropy_backward(record, gradients, None) == code


@pytest.mark.parametrize("softcap", [1e-45, 1e-39, 9e-20])
def test_caps_whose_inverse_may_not_fit_are_refused(lib, softcap):
    """1 / softcap of a subnormal number is infinite, and 0 / softcap then no number."""
    record, at = _cross_entropy(softcap=softcap), 1 << 20
    assert lib.lct_cross_entropy_forward(record, None, 0, None, 0, at, 1 << 40, at, at, None, 0,
                                         None) == E_ARG
    assert lib.lct_cross_entropy_backward(record, _gradients(), None) == E_ARG
