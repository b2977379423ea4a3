"""Train a small language model whose every layer has a gradient here, then decode with it.

    ids -> embedding -> [gated recurrence -> gated feed-forward] x layers -> output projection -> loss

Each layer adds to its input h, in order:

    v, r, i = h Wv^T, h Wr^T, h Wi^T;   h = h + gated_recurrence(v, r, i, decay)
    h = h + gated_feed_forward(h, Wg, Wu, Wd)

and back, with the projections' gradients as plain products:

    dh += gated_feed_forward_grad(...);  dv, dr, di, d_decay = gated_recurrence_grad(..., checkpoints=...)
    dh += dv Wv + dr Wr + di Wi

Rows hold several documents, packed (seq_idx): no state crosses from one to the next.  The gradients go through
clip_grad_norm into float32 buffers for an Adam step on float32 master weights.  Decoding keeps one state per layer:
gated_recurrence's final state after the prompt, then gated_recurrence_update token by token.  A prompt that is cut
out of packed rows takes their seq_idx along, so that each row is continued from its last document alone.

The data are synthetic: a random first-order chain over the vocabulary.

    python examples/train_recurrent_lm.py [--steps 30] [--vocab 4099] [--dim 512] [--layers 2]
"""
import argparse
import math
import os
import sys

import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "mamba2-jax-pallas_b200"))
from mamba2_b200 import (clip_grad_norm, embedding, embedding_grad, gated_feed_forward,  # noqa: E402
                         gated_feed_forward_grad, gated_recurrence, gated_recurrence_grad, gated_recurrence_update,
                         linear_cross_entropy, linear_cross_entropy_grad)

ACT = "silu"


def init(vocab, dim, layers, hidden=None, seed=0, device="cuda"):
    """Float32 parameters by name."""
    hidden = 3 * dim if hidden is None else hidden
    gen = torch.Generator().manual_seed(seed)

    def normal(*shape, std):
        return torch.randn(shape, generator=gen) * std

    p = {"table": normal(vocab, dim, std=1 / math.sqrt(dim)), "head": normal(vocab, dim, std=1 / math.sqrt(dim))}
    for k in range(layers):
        for name in ("v", "r", "i"):
            p[f"{k}.{name}"] = normal(dim, dim, std=1 / math.sqrt(dim))
        # a channel keeps 0.9 to 0.999 of its state where its gate is fully open
        keep = 0.9 + 0.099 * torch.rand(dim, generator=gen)
        p[f"{k}.decay"] = torch.log(torch.expm1(-torch.log(keep) / 8.0))
        p[f"{k}.gate"], p[f"{k}.up"] = (normal(hidden, dim, std=1 / math.sqrt(dim)) for _ in range(2))
        p[f"{k}.down"] = normal(dim, hidden, std=0.5 / math.sqrt(hidden))
    return {k: v.to(device) for k, v in p.items()}


class Model:
    """The model over parameters of one dtype (decay stays float32)."""

    def __init__(self, params, dtype=torch.bfloat16):
        self.p = {k: v if k.endswith("decay") else v.to(dtype) for k, v in params.items()}
        self.layers = sum(k.endswith(".decay") for k in params)
        self.scale = math.sqrt(self.p["table"].shape[1])

    def _mix(self, k, h):
        return tuple(h @ self.p[f"{k}.{n}"].t() for n in ("v", "r", "i")) + (self.p[f"{k}.decay"],)

    def _feed(self, k):
        return self.p[f"{k}.gate"], self.p[f"{k}.up"], self.p[f"{k}.down"]

    def forward(self, ids, seq_idx=None, kept=None, states=None):
        """Hidden states of the last layer; ``kept`` collects what the gradients need, ``states`` the final states."""
        h = embedding(ids, self.p["table"], scale=self.scale)
        for k in range(self.layers):
            mix = self._mix(k, h)
            y, final, points = gated_recurrence(*mix, seq_idx=seq_idx, return_final_state=True, return_checkpoints=True)
            mid = h + y
            if kept is not None:
                kept.append((h, mix, points, mid))
            if states is not None:
                states.append(final)
            h = mid + gated_feed_forward(mid, *self._feed(k), activation=ACT)
        return h

    def loss(self, ids, targets, seq_idx=None):
        return linear_cross_entropy(self.forward(ids, seq_idx), self.p["head"], targets)

    def loss_and_grads(self, ids, targets, seq_idx=None):
        kept = []
        h = self.forward(ids, seq_idx, kept)
        grads = {}
        loss, dh, grads["head"] = linear_cross_entropy_grad(h, self.p["head"], targets)
        for k in reversed(range(self.layers)):
            before, mix, points, mid = kept[k]
            dx, *dw = gated_feed_forward_grad(mid, *self._feed(k), dh, activation=ACT)
            for name, g in zip(("gate", "up", "down"), dw):
                grads[f"{k}.{name}"] = g
            dh = dh + dx
            *dmix, grads[f"{k}.decay"], _ = gated_recurrence_grad(*mix, dh, seq_idx=seq_idx, checkpoints=points)
            rows = before.flatten(0, -2)
            for name, g in zip(("v", "r", "i"), dmix):
                grads[f"{k}.{name}"] = g.flatten(0, -2).t() @ rows
                dh = dh + g @ self.p[f"{k}.{name}"]
        grads["table"] = embedding_grad(ids, dh, self.p["table"].shape[0], scale=self.scale)
        return loss, grads

    def step(self, ids, states):
        """One token per row: hidden states (batch, dim); the states are updated in place."""
        h = embedding(ids, self.p["table"], scale=self.scale)
        for k in range(self.layers):
            _, y = gated_recurrence_update(states[k], *self._mix(k, h), inplace=True)
            h = h + y
            h = h + gated_feed_forward(h, *self._feed(k), activation=ACT)
        return h


def generate(model, prompt, count, seq_idx=None):
    """``count`` ids that continue each row of the prompt, the likeliest first."""
    states, out = [], []
    h = model.forward(prompt, seq_idx, states=states)[:, -1]
    for _ in range(count):
        last = (h @ model.p["head"].t()).argmax(dim=-1)
        out.append(last)
        h = model.step(last, states)
    return torch.stack(out, 1)


def documents(vocab, rows, length, gen):
    """Packed rows of a chain in which each id is followed by one of four: ids, targets, seq_idx."""
    follow = torch.randint(0, vocab, (vocab, 4), generator=gen, device="cuda")

    def draw():
        ids = torch.empty((rows, length + 1), dtype=torch.int64, device="cuda")
        ids[:, 0] = torch.randint(0, vocab, (rows,), generator=gen, device="cuda")
        pick = torch.randint(0, 4, (rows, length), generator=gen, device="cuda")
        ends = torch.rand((rows, length), generator=gen, device="cuda") < 0.02
        fresh = torch.randint(0, vocab, (rows, length), generator=gen, device="cuda")
        for t in range(length):
            ids[:, t + 1] = torch.where(ends[:, t], fresh[:, t], follow[ids[:, t], pick[:, t]])
        targets = torch.where(ends, torch.full_like(fresh, -100), ids[:, 1:])   # nothing foretells a new document
        seq = torch.zeros((rows, length), dtype=torch.int32, device="cuda")
        seq[:, 1:] = torch.cumsum(ends[:, :-1], 1)
        return ids[:, :-1].contiguous(), targets, seq
    return draw


def main(steps=30, vocab=4099, dim=512, layers=2, rows=4, length=256, lr=3e-3, verbose=True):
    gen = torch.Generator(device="cuda").manual_seed(0)
    masters = init(vocab, dim, layers)
    first, second, buffers = ({k: torch.zeros_like(v) for k, v in masters.items()} for _ in range(3))
    draw = documents(vocab, rows, length, gen)
    losses = []
    for step in range(steps):
        loss, grads = Model(masters).loss_and_grads(*draw())
        names = list(masters)
        _, norm = clip_grad_norm([grads[n] for n in names], 1.0, out=[buffers[n] for n in names])
        for n in names:
            g, m, v = buffers[n], first[n], second[n]
            m.lerp_(g, 0.1)
            v.lerp_(g * g, 0.05)
            masters[n].sub_(lr * (m / (1 - 0.9 ** (step + 1))) / ((v / (1 - 0.95 ** (step + 1))).sqrt() + 1e-8))
        losses.append(loss)
        if verbose and step % 5 == 0:
            print(f"step {step:3d}  loss {float(loss):7.4f}  gradient norm {float(norm):8.4f}")
    model = Model(masters)
    ids, targets, seq = draw()
    held_out = model.loss(ids, targets, seq)
    out = generate(model, ids[:, :64].contiguous(), 8, seq[:, :64].contiguous())
    if verbose:
        print(f"held-out loss {float(held_out):.4f}; continuation of row 0: {out[0].tolist()}")
    return torch.stack(losses), held_out, out


if __name__ == "__main__":
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    ap.add_argument("--steps", type=int, default=30)
    ap.add_argument("--vocab", type=int, default=4099)
    ap.add_argument("--dim", type=int, default=512)
    ap.add_argument("--layers", type=int, default=2)
    a = ap.parse_args()
    main(a.steps, a.vocab, a.dim, a.layers)
