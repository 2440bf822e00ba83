"""The attention path's operators together: the layer that keeps its inputs
compressed, the trainer's windowed form, and generation from its model."""
from __future__ import annotations

import attention_oracle as oracle
import pytest
import torch

from examples.nanogpt import train_gpt_lct as trainer
from examples.nanogpt.generate import Generator
from losslessly_compressed_tensors_amd.components import attention, layers
from losslessly_compressed_tensors_amd.tensor_buffer import TensorBuffer

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
SHAPE = {"vocab_size": 512, "num_layers": 2, "model_dim": 256}


def _values(*shape, seed=0):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(
        torch.bfloat16).to(DEV)


def test_window_attention_layer_is_lossless():
    """Compressed and dense saves give the same bits; the gradients of q, k and v
    lie within the attention's own bounds."""
    batch, length, heads, kv_heads, dim = 2, 300, 4, 2, 64
    inputs = [_values(batch, length, h, dim, seed=i) for i, h in enumerate(
        (heads, kv_heads, kv_heads))]
    weight, bias = _values(128, heads * dim, seed=4), torch.zeros(128, device=DEV)
    grad = _values(batch, length, 128, seed=5)
    results = []
    for compressed in (False, True):
        leaves = [t.clone().requires_grad_() for t in inputs]
        w, b = weight.clone().requires_grad_(), bias.clone().requires_grad_()
        buffer = TensorBuffer(32 << 20, device=DEV)
        out = layers.WindowAttention.apply(*(t.transpose(1, 2) for t in leaves), w, b, buffer,
                                           compressed, None, 1024, 100, 3)
        saved = layers.flush_saved()
        assert len(saved) == (4 if compressed else 0)
        out.backward(grad)
        results.append([out.detach(), *(t.grad for t in (*leaves, w, b))])
    assert all(torch.equal(x, y) for x, y in zip(*results))
    q, k, v = (t.transpose(1, 2) for t in inputs)
    grad_attention = (grad.reshape(-1, 128) @ weight).reshape(
        batch, length, heads, dim).transpose(1, 2)
    expected = oracle.attention_with_bounds(q, k, v, oracle.sees(length, length, 100, 3).to(DEV),
                                            layers.ATTENTION_SCALE, grad_attention)
    for got, name in zip(results[0][1:4], ("dq", "dk", "dv")):
        exact, bound = expected[name]
        assert bool(((got.transpose(1, 2).double() - exact).abs() <= bound).all())


def _losses(steps=3, **how):
    model, optimizers = trainer.build(DEV, **SHAPE, **how)
    out = []
    for i in range(steps):
        inputs, targets = trainer.random_tokens(2, 256, DEV, seed=i, token_ids=512)
        out.append(trainer.train_step(model, optimizers, inputs, targets))
    return out, model


def test_trainer_with_window_and_dropout_is_lossless():
    how = dict(window=64, sinks=2, dropout=0.1, compress_weights=False)
    dense, _ = _losses(compress_activations=False, compress_optimizer=False, **how)
    packed, model = _losses(compress_activations=True, compress_optimizer=True, **how)
    assert all(torch.equal(a, b) for a, b in zip(dense, packed))
    assert model.dropout_offset == 3 * 2 * 2
    assert all(bool(loss.isfinite()) for loss in dense)


def test_a_window_of_everything_is_the_trainers_attention():
    """The first losses of the windowed path with all keys visible, without
    dropout, are the default path's within BF16's roundings."""
    plain, _ = _losses(1, compress_weights=False, compress_activations=False,
                       compress_optimizer=False)
    window, _ = _losses(1, compress_weights=False, compress_activations=False,
                        compress_optimizer=False, window=256)
    assert abs(float(plain[0]) - float(window[0])) <= 2.0 ** -8 * abs(float(plain[0]))


def test_generation_follows_the_whole_prompt():
    """Token by token through the caches and as one prompt: the logits agree within
    BF16's roundings, with compressed weights."""
    model, _ = trainer.build(DEV, compress_weights=False, compress_activations=False,
                             compress_optimizer=False, **SHAPE)
    with torch.no_grad():
        for i, p in enumerate(p for name, p in model.named_parameters() if "proj.weight" in name):
            p.copy_(0.05 * _values(*p.shape, seed=i))
    model.set_tensor_buffer(TensorBuffer(32 << 20, device=DEV))
    model.compress_weights()
    tokens = torch.randint(0, 512, (3, 40), generator=torch.Generator().manual_seed(1)).to(DEV)
    whole = Generator(model, 3, 40, window=16, sinks=2).logits(tokens)
    steps = Generator(model, 3, 40, window=16, sinks=2)
    steps.logits(tokens[:, :30])
    for t in range(30, 40):
        last = steps.logits(tokens[:, t:t + 1])
    # Each of 2 layers rounds a dozen times to 2^-8 of values of order one.
    assert float((whole - last).abs().amax()) <= 2 * 12 * 2.0 ** -8 * float(whole.abs().amax())
    out = Generator(model, 3, 48, window=16, sinks=2).generate(tokens, 8)
    assert out.shape == (3, 8) and bool(((out >= 0) & (out < 512)).all())


# The trainer starts from projections of zero, under which nothing of the attention
# reaches a loss: these start from others.


def _started(**how):
    model, optimizers = trainer.build(DEV, compress_weights=False, **SHAPE, **how)
    with torch.no_grad():
        for i, (name, p) in enumerate(model.named_parameters()):
            if name.endswith("proj.weight"):
                p.copy_(0.05 * _values(*p.shape, seed=100 + i))
    return model, optimizers


def _loss_and_gradients(plan=None, **how):
    model, _ = _started(compress_activations=False, compress_optimizer=False, **how)
    if plan is not None:
        for block in model.blocks:
            block.attn.rotary_plan = plan
    inputs, targets = trainer.random_tokens(2, 256, DEV, seed=0, token_ids=512)
    loss = model(inputs, targets)
    loss.backward()
    return float(loss.detach()), {name: p.grad.double() for name, p in model.named_parameters()
                         if ".attn." in name and name.endswith("weight")}


# BF16 rounds a value by 2^-9.8 of it in the mean square; a pass through 2 layers and back
# has some 24 roundings on a path to a gradient, two paths are compared, and twice that.
FAR = 2 * (2 * 2 * 24) ** 0.5 * 2.0 ** -9.8


def test_the_windowed_path_is_the_default_path_under_a_window_of_everything():
    """Loss and the gradients of all of the attention's weights."""
    loss, gradients = _loss_and_gradients()
    same, window = _loss_and_gradients(window=256)
    assert len(gradients) == 2 * 4 and abs(same - loss) <= FAR * abs(loss)
    for name, grad in gradients.items():
        assert float((window[name] - grad).norm()) <= FAR * float(grad.norm()), name
    # What the comparison would not miss: another window, the other sense of rotation,
    # no rotation.
    frequencies = attention.trainer_frequencies(trainer.HEAD_DIM)
    for how in (dict(window=8), dict(window=256, plan=attention.Rotary(-frequencies)),
                dict(window=256, plan=attention.Rotary(0 * frequencies))):
        _, other = _loss_and_gradients(**how)
        assert any(float((other[name] - grad).norm()) > 2 * FAR * float(grad.norm())
                   for name, grad in gradients.items()), how


def test_windowed_training_is_lossless_in_every_parameter():
    """Three steps whose attention gradients are not zero, dense and compressed."""
    results = []
    for compressed in (False, True):
        model, optimizers = _started(compress_activations=compressed,
                                     compress_optimizer=compressed, window=64, sinks=2,
                                     dropout=0.1)
        before = [p.detach().clone() for _, p in model.named_parameters()]
        losses = []
        for i in range(3):
            inputs, targets = trainer.random_tokens(2, 256, DEV, seed=i, token_ids=512)
            losses.append(trainer.train_step(model, optimizers, inputs, targets))
        named = list(model.named_parameters())
        moved = {name for (name, p), old in zip(named, before) if not torch.equal(p, old)}
        assert {name for name, _ in named if ".attn." in name and name.endswith("weight")} <= moved
        results.append(losses + [p.detach() for _, p in named])
    assert all(torch.equal(a, b) for a, b in zip(*results))


def test_generation_begins_with_its_prompts():
    """Again with the same generator, of one token, of none."""
    model, _ = _started(compress_activations=False, compress_optimizer=False)
    prompts = torch.randint(0, 512, (2, 5), generator=torch.Generator().manual_seed(1)).to(DEV)
    generator = Generator(model, 2, 16, window=8)
    for tokens in (prompts, prompts[:, :1]):
        want = Generator(model, 2, 16, window=8).generate(tokens, 4)
        for _ in range(2):
            assert torch.equal(generator.generate(tokens, 4), want)
    with pytest.raises(ValueError, match="steps"):
        generator.generate(prompts, 0)
