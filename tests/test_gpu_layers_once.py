"""The layers' gradients have no derivatives (their saved values come back without a graph): with
``create_graph=True`` they are what they are without it, and a second derivative is an error."""
from __future__ import annotations

import pytest
import torch

from gpu_util import require_gpu
from losslessly_compressed_tensors_amd.components import layers
from losslessly_compressed_tensors_amd.components.ops import rms_norm

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16


@pytest.fixture(autouse=True)
def _gpu():
    require_gpu()


def _inputs(seed=0):
    """A layer's input, a weight, a gain and a bias; queries, keys and values."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(2, 16, 128, generator=g).to(BF16)
    weight = (torch.randn(128, 128, generator=g) / 128 ** 0.5).to(BF16)
    gain, bias = 1 + 0.1 * torch.randn(128, generator=g), torch.randn(128, generator=g)
    heads = [torch.randn(2, 2, 16, 64, generator=g).to(BF16) for _ in range(3)]
    return [t.cuda() for t in (x, weight, gain, bias, *heads)]


def _projection(w, b):
    linear = torch.nn.Module()
    linear.weight, linear.bias = w, b
    return linear


# What each is of, by the inputs' places, and the call.
CALLS = {
    "rms_linear": ((0, 1, 2), lambda x, w, n, b, *_: layers.RMSLinear.apply(x, w, n, b)),
    "qkv": ((0, 1, 2), lambda x, w, n, b, *_: sum(
        layers.rms_norm_qkv(x, n, *[_projection(w, b)] * 3))),
    "rms_norm_function": ((0, 2), lambda x, w, n, *_: layers.RMSNormFunction.apply(
        x, n, None, False, None, 1)),
    "rms_norm": ((0, 2), lambda x, w, n, *_: rms_norm(x, n.to(BF16))[0]),
    "relu2_linear": ((0, 1), lambda x, w, n, b, *_: layers.Relu2Linear.apply(x, w, b)),
    "flash_attention": ((1, 4, 5, 6), lambda x, w, n, b, *qkv: layers.FlashAttention.apply(
        *qkv, w, b, None, False, None, 1)),
    "window_attention": ((1, 4, 5, 6), lambda x, w, n, b, *qkv: layers.WindowAttention.apply(
        *qkv, w, b, None, False, None, 1, 8)),
}


@pytest.mark.parametrize("name", CALLS)
def test_second_derivatives_are_refused(name):
    of, call = CALLS[name]
    for at in of:
        leaves = [t.requires_grad_(i == at) for i, t in enumerate(_inputs())]
        plain, = torch.autograd.grad(call(*leaves).float().sum(), leaves[at])
        grad, = torch.autograd.grad(call(*leaves).float().sum(), leaves[at], create_graph=True)
        assert torch.equal(grad, plain)
        with pytest.raises(RuntimeError, match="differentiated once only"):
            grad.float().square().sum().backward()
