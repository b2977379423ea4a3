"""Cases and plain forms of the language-model operators around the mixer layer.

Five calls are covered: ``embedding`` and ``embedding_grad`` (the model's first step and its
gradient), ``linear_cross_entropy`` and ``linear_cross_entropy_grad`` (output projection and
softmax cross entropy, alone and with both gradients) and ``clip_grad_norm`` (the global norm
over a model's gradients and the scaled gradients for the optimizer).  The widths 768, 2560 and
4096 are those of the benchmark's layers (24, 80 and 128 heads of 64, two inner columns per
model column); vocabularies are generic.
"""
import math
import os
import sys

import numpy as np
import torch

own = False

_DT = {"f32": torch.float32, "bf16": torch.bfloat16}
_IGNORE = -100


def listed():
    return [
        # one decode step of a served batch: 256 requests, one token each
        dict(name="embed decode 256", op="embed", tokens=256, vocab=131072, d=4096, dtype="bf16", skew="zipf"),
        # a training or prefill batch of 8 x 2048 tokens
        dict(name="embed batch 16384", op="embed", tokens=16384, vocab=50000, d=2560, dtype="bf16", skew="zipf"),
        # a short fine-tuning sequence in float32, odd vocabulary
        dict(name="embed grad 777 f32", op="embed_grad", tokens=777, vocab=50257, d=768, dtype="f32", skew="zipf"),
        # the packed 4 x 8192 row of the varlen benchmark, a large vocabulary
        dict(name="embed grad 32768", op="embed_grad", tokens=32768, vocab=131072, d=4096, dtype="bf16", skew="zipf"),
        # scoring a handful of tokens (a drafted continuation, a multiple-choice answer)
        dict(name="loss 7 tokens f32", op="ce", tokens=7, vocab=50257, d=768, dtype="f32", ignored=0.0),
        dict(name="loss 1 token", op="ce", tokens=1, vocab=131072, d=4096, dtype="bf16", ignored=0.0),
        # perplexity of one 4096-token sequence
        dict(name="loss 4096", op="ce", tokens=4096, vocab=131072, d=4096, dtype="bf16", ignored=0.0),
        # one float32 training step of the smallest layer's width
        dict(name="loss grad 2048 f32", op="ce_grad", tokens=2048, vocab=50257, d=768, dtype="f32", ignored=0.0),
        # instruction tuning: most positions are prompt and carry no loss; odd sizes
        dict(name="loss grad 3001 ragged", op="ce_grad", tokens=3001, vocab=32003, d=1000, dtype="bf16", ignored=0.7),
        # the training batch of 8 x 2048 tokens
        dict(name="loss grad 16384", op="ce_grad", tokens=16384, vocab=50000, d=2560, dtype="bf16", ignored=0.0),
        # many small tensors: a narrow 24-layer model
        dict(name="clip narrow f32", op="clip", layers=24, d=64, vocab=0, dtype="f32", out="f32"),
        # 24 wide layers and an embedding, bf16 gradients into the optimizer's float32 buffers
        dict(name="clip wide bf16", op="clip", layers=24, d=2560, vocab=50000, dtype="bf16", out="f32"),
    ]


def _log(rng, lo, hi):
    n = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    n = min(max(n, lo), hi)
    return n + 1 if n == 3072 else n


def draw(rng):
    op = rng.choice(["embed", "embed_grad", "ce", "ce_grad", "ce_grad", "clip"])
    if op == "clip":
        d = 64 * rng.choice([k for k in range(1, 41) if k not in (24, 48)])
        return dict(op=op, layers=rng.randint(1, 24), d=d, vocab=rng.choice([0, _log(rng, 100, 50000)]),
                    dtype=rng.choice(["f32", "bf16"]), out=rng.choice(["f32", "bf16"]))
    dtype = rng.choice(["f32", "bf16"])
    d = _log(rng, 64, 4096)
    if rng.random() < 0.6:
        d = max(64, d // 64 * 64)
        d += 64 * (d == 3072)
    vocab = _log(rng, 500, 131072)
    if op in ("embed", "embed_grad"):
        return dict(op=op, tokens=_log(rng, 1, 32768), vocab=vocab, d=d, dtype=dtype,
                    skew=rng.choice(["zipf", "zipf", "uniform", "one"]))
    most = 16384 * 50000 * 2560 // (vocab * d) // (4 if dtype == "f32" else 1)
    tokens = _log(rng, 1, min(16384, max(1, most)))
    return dict(op=op, tokens=tokens, vocab=vocab, d=d, dtype=dtype,
                ignored=rng.choice([0.0, 0.0, 0.2, 0.7, 0.97]) if tokens >= 200 else 0.0)


def _grad_shapes(case):
    """Gradient shapes of a Mamba2 language model: the layer's parameters and, with a vocabulary, its table."""
    d, di = case["d"], 2 * case["d"]
    conv, heads = di + 2 * 128, di // 64
    layer = [(d, 2 * di + 2 * 128 + heads), (di, d), (conv, 4), (conv,), (heads,), (heads,), (heads,), (di,), (d,)]
    return layer * case["layers"] + [(d,)] + ([(case["vocab"], d)] if case["vocab"] else [])


def _ids(case, gen, n):
    """Token ids: about Zipf's law (log-uniform ranks), uniform, or a single id."""
    u = torch.rand(n, generator=gen, device="cuda")
    v = case["vocab"]
    skew = case.get("skew", "zipf")
    if skew == "one":
        return torch.full((n,), int(float(u[0]) * (v - 1)), dtype=torch.int64, device="cuda")
    ids = u * v if skew == "uniform" else torch.exp(u * math.log(v)) - 1
    return ids.to(torch.int64).clamp_(0, v - 1)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dt = _DT[case["dtype"]]

    def normal(*shape):
        return torch.randn(shape, generator=gen, device="cuda")

    st = dict(case=case)
    if case["op"] == "clip":
        # per-tensor scales as in training: some layers' gradients are much larger than others'
        shapes = _grad_shapes(case)
        scale = torch.exp(torch.randn(len(shapes), generator=gen, device="cuda") - 5.0)
        st["grads"] = [(normal(*s) * scale[i]).to(dt) for i, s in enumerate(shapes)]
        # the optimizer keeps one flat buffer; each parameter has its piece of it
        st["flat"] = torch.empty(sum(math.prod(s) for s in shapes), dtype=_DT[case["out"]], device="cuda")
        pieces = torch.split(st["flat"], [math.prod(s) for s in shapes])
        st["out"] = [p.view(s) for p, s in zip(pieces, shapes)]
        st["max_norm"] = 1.0
        return st
    t, v, d = case["tokens"], case["vocab"], case["d"]
    ids = _ids(case, gen, t)
    if case["op"] == "embed":
        st.update(tokens=ids, weight=normal(v, d).mul_(0.02).to(dt), scale=math.sqrt(d))
    elif case["op"] == "embed_grad":
        st.update(tokens=ids, grad=normal(t, d).mul_(1e-3).to(dt), scale=math.sqrt(d))
    else:
        weight = normal(v, d).mul_(1.0 / math.sqrt(d)).to(dt)
        # a trained model: some tokens are predicted with confidence, others not at all
        gain = torch.rand(t, 1, generator=gen, device="cuda") * 14.0
        hidden = (normal(t, d) + gain * weight[ids].float()).to(dt)
        if case["ignored"]:
            drop = torch.rand(t, generator=gen, device="cuda") < case["ignored"]
            ids = torch.where(drop, torch.full_like(ids, _IGNORE), ids)
        st.update(hidden=hidden, weight=weight, targets=ids)
    return st


def _ops():
    root = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "mamba2-jax-pallas_b200")
    if root not in sys.path:
        sys.path.insert(0, root)
    import mamba2_b200
    return mamba2_b200


def _run_own(st):
    m, case = _ops(), st["case"]
    op = case["op"]
    if op == "embed":
        return m.embedding(st["tokens"], st["weight"], scale=st["scale"])
    if op == "embed_grad":
        return m.embedding_grad(st["tokens"], st["grad"], case["vocab"], scale=st["scale"])
    if op == "ce":
        # the losses of the single positions: what a perplexity or a score is made of
        return m.linear_cross_entropy(st["hidden"], st["weight"], st["targets"], reduction="none")
    if op == "ce_grad":
        return m.linear_cross_entropy_grad(st["hidden"], st["weight"], st["targets"], reduction="mean")
    _, norm = m.clip_grad_norm(st["grads"], st["max_norm"], out=st["out"])
    return st["flat"], norm


def run(st):
    if own:
        return _run_own(st)
    case = st["case"]
    op, dt = case["op"], _DT[case["dtype"]]
    if op == "embed":
        return (st["weight"][st["tokens"]].float() * st["scale"]).to(dt)
    if op == "embed_grad":
        g = st["grad"].float() * st["scale"]
        return torch.zeros(case["vocab"], case["d"], device=g.device).index_add_(0, st["tokens"], g).to(dt)
    if op == "clip":
        flat = torch.cat([g.reshape(-1).float() for g in st["grads"]])
        norm = torch.sqrt((flat * flat).sum())
        coef = torch.clamp(st["max_norm"] / (norm + 1e-6), max=1.0)
        return (flat * coef).to(_DT[case["out"]]), norm
    x, w, y = st["hidden"].float(), st["weight"].float(), st["targets"]
    logits = x @ w.t()
    top = logits.max(dim=1, keepdim=True).values
    e = torch.exp(logits - top)
    total = e.sum(dim=1, keepdim=True)
    valid = y != _IGNORE
    col = torch.where(valid, y, torch.zeros_like(y))[:, None]
    loss = torch.where(valid, (torch.log(total) + (top - logits.gather(1, col)))[:, 0], torch.zeros_like(top[:, 0]))
    if op == "ce":
        return loss
    coef = valid.float()[:, None] / valid.sum().clamp(min=1).float()
    dl = e * (coef / total)
    dl.scatter_add_(1, col, -coef)
    return loss.sum() * (1.0 / valid.sum().clamp(min=1).float()), (dl @ w).to(dt), (dl.t() @ x).to(dt)


def _rows_named(case):
    """Table rows that the ids of a case are expected to name (each is read once)."""
    t, v = case["tokens"], case["vocab"]
    if case["skew"] == "one":
        return 1
    rank = np.arange(1.0, v + 1)
    p = np.full(v, 1.0 / v) if case["skew"] == "uniform" else np.log1p(1.0 / rank) / np.log(v + 1.0)
    return max(1, round(float(-np.expm1(t * np.log1p(-p)).sum())))


def work(case):
    es = 4 if case["dtype"] == "f32" else 2
    if case["op"] == "clip":
        n = sum(math.prod(s) for s in _grad_shapes(case))
        return {"bytes": n * (es + (4 if case["out"] == "f32" else 2)), "flops": 3 * n}
    t, v, d = case["tokens"], case["vocab"], case["d"]
    if case["op"] == "embed":
        return {"bytes": (_rows_named(case) + t) * d * es + 8 * t, "flops": t * d}
    if case["op"] == "embed_grad":
        return {"bytes": t * d * es + v * d * es + 8 * t, "flops": 2 * t * d}
    counted = max(1, round(t * (1 - case["ignored"])))  # an ignored position needs no logits
    if case["op"] == "ce":
        return {"bytes": (counted + v) * d * es + 8 * t + 4 * t, "flops": 2 * counted * v * d}
    return {"bytes": (counted + t + 2 * v) * d * es + 8 * t + 4, "flops": 6 * counted * v * d}


def exact(case, seed):
    st = prepare(case, seed)
    f64 = torch.float64
    if case["op"] == "clip":
        sq = torch.stack([torch.linalg.vector_norm(g.to(f64)) for g in st["grads"]])
        norm = torch.linalg.vector_norm(sq)
        c = min(1.0, st["max_norm"] / (float(norm) + 1e-6))
        return torch.cat([g.to(f64).mul_(c).flatten() for g in st["grads"]]), norm
    if case["op"] == "embed":
        return torch.index_select(st["weight"], 0, st["tokens"]).to(f64) * st["scale"]
    if case["op"] == "embed_grad":
        table = torch.zeros(case["vocab"], case["d"], dtype=f64, device="cuda")
        for lo in range(0, case["tokens"], 4096):
            table.index_add_(0, st["tokens"][lo:lo + 4096], st["grad"][lo:lo + 4096].to(f64))
        return table * st["scale"]
    w = st["weight"].to(f64)
    losses, dx, dw = [], [], torch.zeros_like(w) if case["op"] == "ce_grad" else None
    n = max(1, int((st["targets"] >= 0).sum()))
    for lo in range(0, case["tokens"], 2048):
        x, y = st["hidden"][lo:lo + 2048].to(f64), st["targets"][lo:lo + 2048]
        logp = torch.log_softmax(x @ w.T, dim=-1)
        on = (y >= 0).to(f64)
        rows, picked = torch.arange(len(y), device="cuda"), y.clamp(min=0)
        losses.append(-logp[rows, picked] * on)
        if dw is not None:
            p = logp.exp_()
            p[rows, picked] -= 1.0
            p *= on[:, None] / n
            dx.append(p @ w)
            dw += p.T @ x
    loss = torch.cat(losses)
    return loss if dw is None else (loss.sum() / n, torch.cat(dx), dw)
