"""Adapt the two ends of a language model around frozen Mamba2 layers.

    ids -> embedding (trained) + features of the frozen backbone -> output projection (trained) -> loss

The backbone is a stack of mixer layers over its own frozen copy of the token table, so its
output does not depend on what is trained and the gradients below are exact:

    h = scale * E[ids] + backbone(ids)          embedding
    loss, dh, dW                                linear_cross_entropy_grad
    dE = embedding_grad(ids, dh)                embedding_grad
    gradients -> float32, norm at most 1        clip_grad_norm
    Adam step on float32 master weights

Then the adapted model scores a held-out row (linear_cross_entropy) and continues a prompt token
by token (embedding of single tokens, the layers' decode step).

The data are synthetic: a random first-order chain over the vocabulary, which the trained ends
can learn and the random backbone does not know.

    python examples/adapt_lm_ends.py [--steps 30] [--vocab 4099] [--d-model 512] [--layers 2]
"""
import argparse
import math
import os
import sys

import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "mamba2-jax-pallas_b200"))
from mamba2_b200 import (clip_grad_norm, embedding, embedding_grad, linear_cross_entropy,  # noqa: E402
                         linear_cross_entropy_grad)
from mamba2_b200.modules import Mamba2, allocate_inference_cache  # noqa: E402


class Backbone:
    """Frozen token table and residual mixer layers."""

    def __init__(self, table, d_model, n_layers):
        self.table, self.scale = table, math.sqrt(d_model)
        self.layers = [Mamba2(d_model=d_model, ngroups=2, chunk_size=128, seed=i) for i in range(n_layers)]

    def __call__(self, ids):
        h = embedding(ids, self.table, scale=self.scale)
        for layer in self.layers:
            h = h + layer(h)
        return h

    def prefill(self, ids):
        h = embedding(ids, self.table, scale=self.scale)
        caches = []
        for layer in self.layers:
            out, cache = layer(h, inference_params=allocate_inference_cache(ids.shape[0], layer))
            h, caches = h + out, caches + [cache]
        return h, caches

    def step(self, ids, caches):
        h = embedding(ids, self.table, scale=self.scale)
        for i, layer in enumerate(self.layers):
            out, caches[i] = layer(h, inference_params=caches[i])
            h = h + out
        return h, caches


def chain(vocab, rows, length, gen):
    """Rows of a chain in which each id is followed by one of four."""
    follow = torch.randint(0, vocab, (vocab, 4), generator=gen, device="cuda")

    def draw():
        ids = torch.empty((rows, length + 1), dtype=torch.int64, device="cuda")
        ids[:, 0] = torch.randint(0, vocab, (rows,), generator=gen, device="cuda")
        pick = torch.randint(0, 4, (rows, length), generator=gen, device="cuda")
        for t in range(length):
            ids[:, t + 1] = follow[ids[:, t], pick[:, t]]
        return ids
    return draw


def main(steps=30, vocab=4099, d_model=512, n_layers=2, rows=4, length=256, lr=5e-3, verbose=True):
    gen = torch.Generator(device="cuda").manual_seed(0)
    bf = torch.bfloat16
    table = torch.randn((vocab, d_model), generator=gen, device="cuda") / math.sqrt(d_model)
    backbone = Backbone(table.to(bf), d_model, n_layers)
    # trained weights: float32 masters, bfloat16 copies for the kernels
    masters = [table.clone(), torch.randn((vocab, d_model), generator=gen, device="cuda") / d_model]
    first, second = ([torch.zeros_like(m) for m in masters] for _ in range(2))
    buffers = [torch.empty_like(m) for m in masters]
    scale = math.sqrt(d_model)
    draw = chain(vocab, rows, length, gen)
    losses = []
    for step in range(steps):
        ids = draw()
        x, y = ids[:, :-1].contiguous(), ids[:, 1:].clone()
        y[:, : length // 8] = -100          # a prompt that carries no loss
        e, w = (m.to(bf) for m in masters)
        h = embedding(x, e, scale=scale) + backbone(x)
        loss, dh, dw = linear_cross_entropy_grad(h, w, y)
        de = embedding_grad(x, dh, vocab, scale=scale)
        grads, norm = clip_grad_norm([de, dw], 1.0, out=buffers)
        for p, m, v, g in zip(masters, first, second, grads):
            m.lerp_(g, 0.1)
            v.lerp_(g * g, 0.05)
            p.sub_(lr * (m / (1 - 0.9 ** (step + 1))) / ((v / (1 - 0.95 ** (step + 1))).sqrt() + 1e-8))
        losses.append(loss)
        if verbose and step % 5 == 0:
            print(f"step {step:3d}  loss {float(loss):7.4f}  gradient norm {float(norm):8.4f}")
    e, w = (m.to(bf) for m in masters)
    ids = draw()
    x, y = ids[:, :-1].contiguous(), ids[:, 1:].contiguous()
    held_out = linear_cross_entropy(embedding(x, e, scale=scale) + backbone(x), w, y)
    # continue a prompt: prefill, then single tokens
    prompt = x[:, :128].contiguous()
    h, caches = backbone.prefill(prompt)
    last = prompt[:, -1:]
    h = h[:, -1:] + embedding(last, e, scale=scale)
    out = []
    for _ in range(8):
        last = (h[:, -1] @ w.t()).argmax(dim=-1, keepdim=True)
        out.append(last)
        f, caches = backbone.step(last, caches)
        h = embedding(last, e, scale=scale) + f
    if verbose:
        print(f"held-out loss {float(held_out):.4f}; continuation of row 0: {torch.cat(out, 1)[0].tolist()}")
    return torch.stack(losses), held_out, torch.cat(out, 1)


if __name__ == "__main__":
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    ap.add_argument("--steps", type=int, default=30)
    ap.add_argument("--vocab", type=int, default=4099)
    ap.add_argument("--d-model", type=int, default=512)
    ap.add_argument("--layers", type=int, default=2)
    a = ap.parse_args()
    main(a.steps, a.vocab, a.d_model, a.layers)
