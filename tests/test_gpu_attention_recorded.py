"""The attention path's public calls where something has to see their operations:
an error, and caches as they were."""
from __future__ import annotations

import pytest
import torch
from torch.autograd import forward_ad

from losslessly_compressed_tensors_amd.components import attention, layers
from losslessly_compressed_tensors_amd.components.dropout import dropout_add

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _values(*shape, seed=0):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).bfloat16().to(DEV)


def _calls():
    plan = attention.Rotary(attention.rotary_frequencies(64))
    heads, token, cache = _values(1, 2, 9, 64), _values(1, 2, 64), _values(1, 9, 2, 64)
    at = torch.tensor([4], dtype=torch.int32, device=DEV)
    weight, bias = _values(32, 128), torch.zeros(32, device=DEV)
    return {
        "window": (lambda t: attention.window_attention(t, heads, heads, window=3), heads),
        "layer": (lambda t: layers.WindowAttention.apply(t, heads, heads, weight, bias, None, False,
                                                         None, 0, 3), heads),
        "decode": (lambda t: attention.decode_attention(t, cache, cache, at), token),
        "rotary": (lambda t: attention.apply_rotary(plan, t), cache),
        "append": (lambda t: attention.rotary_append(plan, t, token, token, cache, cache.clone(),
                                                     at), token),
        "dropout": (lambda t: dropout_add(t, heads, 0.5, 3), heads)}, cache


@pytest.mark.filterwarnings("ignore::DeprecationWarning", "ignore::torch.jit.TracerWarning")
def test_public_calls_are_refused():
    calls, cache = _calls()
    before = cache.clone()
    for call, tensor in calls.values():
        for leaf in (tensor, tensor.clone().requires_grad_()):
            with pytest.raises(RuntimeError, match="recorded|gradient"):
                try:
                    torch.jit.trace(call, (leaf,), check_trace=False)
                except ValueError as error:      # append and decode of a leaf
                    raise RuntimeError(str(error)) from error
        with forward_ad.dual_level():
            with pytest.raises(RuntimeError):
                call(forward_ad.make_dual(tensor, torch.ones_like(tensor)))
            call(tensor)                         # no tangent: as ever
    # Only the last call of the append, outside a trace, wrote.
    assert torch.equal(cache[:, 5:], before[:, 5:]) and torch.equal(cache[:, :4], before[:, :4])


def test_a_gradient_with_a_tangent_is_refused():
    heads = _values(1, 2, 9, 64).requires_grad_()
    out = attention.window_attention(heads, heads, heads)
    with forward_ad.dual_level(), pytest.raises(RuntimeError):
        torch.autograd.grad(out, heads, forward_ad.make_dual(torch.ones_like(out),
                                                             torch.ones_like(out)))
