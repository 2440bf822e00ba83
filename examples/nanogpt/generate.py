"""Generation from the trainer's model with its weights held compressed.

The reference has no serving form.  Here a prompt runs through windowed attention
and fills a cache per layer (``components/attention.py``'s ``KVCache``), then every
new token takes, per layer, one launch that turns its query and key and writes
the caches, and one or two of attention over them; the projections are
``A_compBT`` products with the compressed weights.  The arithmetic is the
trainer's (``train_gpt_lct.py``): RMS-normalised queries and keys, half-truncated
rotary frequencies, attention scale 0.12, squared ReLU, soft-capped logits.

``python examples/nanogpt/generate.py --window 256 --sinks 4`` prints the tokens
per second of random-weight generation.
"""
from __future__ import annotations

import argparse
import json
import sys
import time
from pathlib import Path

if __package__ in (None, ""):
    sys.path.insert(0, str(Path(__file__).resolve().parents[2]))

import torch
import torch.nn.functional as F
from torch import Tensor

from examples.nanogpt.train_gpt_lct import (
    HEAD_DIM, MODEL_DIM, NUM_LAYERS, SOFTCAP, TOKEN_IDS, VOCAB_SIZE, build,
)
from losslessly_compressed_tensors_amd.LCTensor import LCTTensor
from losslessly_compressed_tensors_amd.components.attention import KVCache, window_attention
from losslessly_compressed_tensors_amd.components.layers import ATTENTION_SCALE, dense_weight
from losslessly_compressed_tensors_amd.components.ops import rms_norm
from losslessly_compressed_tensors_amd.operations import A_compBT


def _project(x: Tensor, module) -> Tensor:
    """``module``'s projection of [.., channels]; few rows against a compressed
    weight go through ``A_compBT``."""
    rows = x.reshape(-1, x.shape[-1])
    if isinstance(module.weight, LCTTensor):
        out = A_compBT(rows, module.weight.x)
    else:
        out = rows @ module.weight.T
    return (out + module.bias.to(out.dtype)).view(*x.shape[:-1], -1)


def _normed(x: Tensor, gains: Tensor | None) -> Tensor:
    return rms_norm(x, None if gains is None else gains.to(x.dtype))[0]


class Generator:
    """One model's caches for ``batch`` sequences of up to ``capacity`` tokens."""

    def __init__(self, model, batch: int, capacity: int, window: int | None = None,
                 sinks: int = 0):
        self.model, self.window, self.sinks = model, window, sinks
        device = model.norm1.gains.device
        self.caches = [KVCache(batch, capacity, block.attn.num_heads, block.attn.head_dim,
                               device=device) for block in model.blocks]

    def _block(self, block, cache, x: Tensor) -> Tensor:
        """[batch, token, channels]: all tokens of the prompts, or one of each."""
        attn = block.attn
        batch, tokens = x.shape[:2]
        shape = (batch, tokens, attn.num_heads, attn.head_dim)
        normed = _normed(x, block.norm1.gains)
        q, k, v = (_project(normed, m).view(shape) for m in (attn.q, attn.k, attn.v))
        q, k, plan = _normed(q, None), _normed(k, None), attn.plan(x.device)
        how = {"window": self.window, "sinks": self.sinks, "scale": ATTENTION_SCALE}
        if tokens > 1:
            q, k = cache.fill(plan, q, k, v)
            hidden = window_attention(q.transpose(1, 2), k.transpose(1, 2), v.transpose(1, 2),
                                      **how).transpose(1, 2)
        else:
            hidden = cache.attend(cache.append(plan, q[:, 0], k[:, 0], v[:, 0]), **how)
        x = x + _project(hidden.reshape(batch, tokens, -1), attn.proj)
        z = _project(_normed(x, block.norm2.gains), block.mlp.fc)
        return x + _project(z.relu().square(), block.mlp.proj)

    @torch.no_grad()
    def logits(self, tokens: Tensor) -> Tensor:
        """[batch, vocabulary] after ``tokens`` [batch, n]: prompts (n > 1, into empty
        caches), or the next token of each sequence (n = 1)."""
        model = self.model
        x = _normed(F.embedding(tokens, dense_weight(model.embed.weight)), model.norm1.gains)
        for block, cache in zip(model.blocks, self.caches):
            x = self._block(block, cache, x)
        last = _project(_normed(x[:, -1], model.norm2.gains), model.proj).float()
        return SOFTCAP * last * (last.square() + SOFTCAP ** 2).rsqrt()

    def generate(self, prompts: Tensor, steps: int) -> Tensor:
        """The ``steps`` likeliest tokens after each prompt, [batch, steps]."""
        if steps < 1:
            raise ValueError("steps must be at least 1")
        for cache in self.caches:
            cache.reset()
        token = self.logits(prompts).argmax(-1)
        out = [token]
        for _ in range(steps - 1):
            token = self.logits(token.unsqueeze(1)).argmax(-1)
            out.append(token)
        return torch.stack(out, 1)


def main():
    parser = argparse.ArgumentParser(description=__doc__.split("\n")[0])
    parser.add_argument("--batch", type=int, default=8)
    parser.add_argument("--prompt", type=int, default=512)
    parser.add_argument("--steps", type=int, default=64)
    parser.add_argument("--layers", type=int, default=NUM_LAYERS)
    parser.add_argument("--window", type=int, default=None)
    parser.add_argument("--sinks", type=int, default=0)
    args = parser.parse_args()
    if not torch.cuda.is_available():
        raise RuntimeError("generation needs a GPU")
    device = torch.device("cuda:0")
    model, _ = build(device, compress_weights=True, compress_activations=False,
                     compress_optimizer=False, vocab_size=VOCAB_SIZE, num_layers=args.layers,
                     model_dim=MODEL_DIM, head_dim=HEAD_DIM)
    prompts = torch.randint(0, TOKEN_IDS, (args.batch, args.prompt), device=device)
    for timed in (False, True):
        generator = Generator(model, args.batch, args.prompt + args.steps, args.window, args.sinks)
        torch.cuda.synchronize()
        start = time.perf_counter()
        generator.generate(prompts, args.steps)
        torch.cuda.synchronize()
        if timed:
            elapsed = time.perf_counter() - start
            print(json.dumps({"tokens_per_s": round(args.batch * args.steps / elapsed, 1),
                              "ms_per_step": round(1e3 * elapsed / args.steps, 3)}), flush=True)


if __name__ == "__main__":
    main()
