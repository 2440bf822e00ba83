"""CPU: what has to see the attention path's launches (a trace, a dispatch mode,
forward-mode differentiation) gets an error, not an unwritten result."""
from __future__ import annotations

import pytest
import torch
from torch._subclasses import FakeTensorMode
from torch.autograd import forward_ad
from torch.fx.experimental.proxy_tensor import make_fx
from torch.utils._python_dispatch import TorchDispatchMode

from losslessly_compressed_tensors_amd.components import attention
from losslessly_compressed_tensors_amd.kernels import attention as kernels

PLAN = attention.Rotary([1.0, 0.5], device="cpu")
LENGTHS = torch.tensor([3], dtype=torch.int32)


def _values(*shape, seed=0):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).bfloat16()


HEADS = _values(1, 2, 3, 8)                 # [batch, head, token, channel]
TOKEN = _values(1, 2, 8, seed=1)            # [batch, head, channel]
CACHE = _values(1, 3, 2, 8, seed=2)         # [batch, token, head, channel]
LSE = torch.zeros(256)

# Each launch as a function of one tensor, and that tensor.
LAUNCHES = {
    "forward": (lambda t: kernels.attention_forward(t, HEADS, HEADS, 0, 0, 0.3, None, True)[0],
                HEADS),
    "forward of v": (lambda t: kernels.attention_forward(HEADS, HEADS, t, 0, 0, 0.3, None, True)[0],
                     HEADS),
    "backward": (lambda t: kernels.attention_backward(t, HEADS, HEADS, HEADS, HEADS, LSE, 0, 0, 0.3,
                                                      None)[0], HEADS),
    "decode": (lambda t: kernels.attention_decode(t, CACHE, CACHE, 0, 0, 0.3, LENGTHS), TOKEN),
    "decode of a cache": (lambda t: kernels.attention_decode(TOKEN, CACHE, t, 0, 0, 0.3, LENGTHS),
                          CACHE),
    "rotate": (lambda t: kernels.rotate(PLAN, t, None, None, 0, False)[0], CACHE),
    "rotate of k": (lambda t: kernels.rotate(PLAN, CACHE, t, None, 0, False)[1], CACHE),
    "append": (lambda t: kernels.rotate_into(PLAN, t, TOKEN, TOKEN, CACHE, CACHE, LENGTHS), TOKEN),
    "append of v": (lambda t: kernels.rotate_into(PLAN, TOKEN, TOKEN, t, CACHE, CACHE, LENGTHS),
                    TOKEN),
    "dropout": (lambda t: kernels.dropout(t, None, 100, 1, 2, None), HEADS),
    "dropout of the residual": (lambda t: kernels.dropout(HEADS, t, 100, 1, 2, None), HEADS),
}


@pytest.fixture(params=LAUNCHES, ids=str)
def launch(request, monkeypatch):
    """``(call, tensor, launches)``; the launches themselves only leave a mark."""
    done = []
    monkeypatch.setattr(kernels, "_launch", lambda name, *a: done.append(name))
    return (*LAUNCHES[request.param], done)


class _Mode(TorchDispatchMode):
    def __torch_dispatch__(self, func, types, args=(), kwargs=None):
        return func(*args, **(kwargs or {}))


def test_a_plain_call_launches(launch):
    call, tensor, done = launch
    call(tensor)
    assert len(done) == 1
    with forward_ad.dual_level():           # no input has a tangent
        call(tensor)
    assert len(done) == 2


@pytest.mark.filterwarnings("ignore::DeprecationWarning")
def test_a_trace_is_refused(launch):
    call, tensor, done = launch
    with pytest.raises(RuntimeError, match="recorded"):
        torch.jit.trace(call, (tensor,), check_trace=False)
    assert not done


@pytest.mark.filterwarnings("ignore::DeprecationWarning")
def test_a_graph_of_operations_is_refused(launch):
    call, tensor, done = launch
    with pytest.raises(RuntimeError, match="recorded"):
        make_fx(call)(tensor)
    assert not done


def test_a_dispatch_mode_is_refused(launch):
    call, tensor, done = launch
    with _Mode(), pytest.raises(RuntimeError, match="recorded"):
        call(tensor)
    assert not done


def test_a_tangent_is_refused(launch):
    call, tensor, done = launch
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(tensor, torch.ones_like(tensor))
        for grad in (True, False):
            with torch.set_grad_enabled(grad), pytest.raises(RuntimeError, match="forward-mode"):
                call(dual)
    assert not done


def test_index_tensors_without_memory_are_refused():
    """Their address of zero would mean that there are none."""
    fake = FakeTensorMode().from_tensor(LENGTHS)
    zero = torch._efficientzerotensor((1,), dtype=torch.int32)
    for t in (fake, zero):
        with pytest.raises(TypeError, match="plain"):
            attention._indices(t, "lengths", ((1,),), t.device)
    assert attention._indices(LENGTHS, "lengths", ((1,),), LENGTHS.device) is LENGTHS
    with pytest.raises(TypeError, match="Tensor"):
        attention._indices(3, "lengths", ((1,),), LENGTHS.device)
    torch.func.vmap(lambda t: _wrapped_is_refused(t))(torch.zeros(2, 1, dtype=torch.int32))


def _wrapped_is_refused(t):
    with pytest.raises(TypeError, match="plain"):
        attention._indices(t, "lengths", ((1,),), t.device)
    return t
