"""Cases and plain forms of the trainable block operators: a gated linear recurrence and a gated feed-forward block.

``gated_recurrence`` carries one state per channel along the sequence,

    a = exp(-scale softplus(decay) sigmoid(decay_gate)),   h = a h + sqrt(1 - a^2) sigmoid(input_gate) x,

over whole sequences, packed rows, with its gradients, and for single tokens
(``gated_recurrence_update``).  ``gated_feed_forward`` is ``(act(x Wg^T) * (x Wu^T)) Wd^T`` with its
gradients.  The widths 768, 2560 and 4096 are those of the benchmark's layers (inner widths twice
that); feed-forward widths are generic.
"""
import math
import os
import sys

import torch

own = False

_DT = {"f32": torch.float32, "bf16": torch.bfloat16}
_SCALE = 8.0


def listed():
    return [
        # one decode step of a served batch: 256 requests, one token each
        dict(name="recurrence step 256", op="rec_step", batch=256, d=8192, dtype="bf16"),
        # a short float32 batch of odd sizes
        dict(name="recurrence 3x777 f32", op="rec", batch=3, length=777, d=1000, dtype="f32", seqs=1),
        # prefill of one prompt
        dict(name="recurrence 4096", op="rec", batch=1, length=4096, d=4096, dtype="bf16", seqs=1),
        # the packed 4 x 8192 row of the varlen benchmark: 16 sequences
        dict(name="recurrence packed 32768", op="rec", batch=1, length=32768, d=5120, dtype="bf16", seqs=16),
        # the training batch of 8 x 2048 tokens: forward, then backward
        dict(name="recurrence train 8x2048", op="rec_train", batch=8, length=2048, d=5120, dtype="bf16", seqs=1),
        # one long document, few channels: backward alone (the forward's values were not kept)
        dict(name="recurrence grad 65536", op="rec_grad", batch=1, length=65536, d=1536, dtype="bf16", seqs=1),
        # one token of one request
        dict(name="feed-forward 1", op="ff", tokens=1, d=4096, f=12288, dtype="bf16", act="silu"),
        # a drafted continuation in float32
        dict(name="feed-forward 7 f32", op="ff", tokens=7, d=768, f=2048, dtype="f32", act="gelu"),
        # a prefill of odd sizes: rows that start at no 16-byte boundary
        dict(name="feed-forward 777 odd", op="ff", tokens=777, d=1001, f=2731, dtype="bf16", act="silu"),
        # prefill of one 4096-token prompt
        dict(name="feed-forward 4096", op="ff", tokens=4096, d=4096, f=12288, dtype="bf16", act="silu"),
        # one float32 training step of the smallest layer's width: backward
        dict(name="feed-forward grad 2048 f32", op="ff_grad", tokens=2048, d=768, f=2048, dtype="f32", act="gelu_tanh"),
        # the training batch of 8 x 2048 tokens: backward
        dict(name="feed-forward grad 16384", op="ff_grad", tokens=16384, d=2560, f=7680, dtype="bf16", act="silu"),
    ]


def _log(rng, lo, hi):
    n = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    return min(max(n, lo), hi)


def _width(rng, lo, hi):
    """Mostly multiples of 64, otherwise any number."""
    n = _log(rng, lo, hi)
    return max(64, n // 64 * 64) if rng.random() < 0.7 else n


def draw(rng):
    op = rng.choice(["rec_step", "rec", "rec", "rec_train", "rec_grad", "ff", "ff", "ff_grad", "ff_grad"])
    dtype = rng.choice(["bf16", "bf16", "f32"])
    if op == "rec_step":
        return dict(op=op, batch=_log(rng, 1, 512), d=_width(rng, 64, 8192), dtype=dtype)
    if op.startswith("rec"):
        d = _width(rng, 64, 8192)
        length = _log(rng, 1, 65536)
        most = max(1, 100_000_000 // (d * length))
        return dict(op=op, batch=_log(rng, 1, min(64, most)), length=length, d=d, dtype=dtype,
                    seqs=rng.choice([1, 1, 1, 3, 16]) if length >= 64 else 1)
    d = _width(rng, 64, 4096)
    f = _width(rng, 64, 12288)
    most = 16384 * 2560 * 7680 // (d * f) // (6 if dtype == "f32" else 1)
    return dict(op=op, tokens=_log(rng, 1, min(16384, max(1, most))), d=d, f=f, dtype=dtype,
                act=rng.choice(["silu", "gelu", "gelu_tanh", "relu"]))


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dt = _DT[case["dtype"]]
    d = case["d"]

    def normal(*shape, scale=1.0):
        return torch.randn(shape, generator=gen, device="cuda").mul_(scale).to(dt)

    st = dict(case=case)
    if case["op"].startswith("ff"):
        t, f = case["tokens"], case["f"]
        st.update(x=normal(t, d), w_gate=normal(f, d, scale=1 / math.sqrt(d)), w_up=normal(f, d, scale=1 / math.sqrt(d)),
                  w_down=normal(d, f, scale=1 / math.sqrt(f)))
        if case["op"] == "ff_grad":
            st["grad"] = normal(t, d, scale=1e-3)
        return st
    # a layer keeps between 0.9 and 0.999 of its state where the gate is fully open, as such layers start out
    keep = 0.9 + 0.099 * torch.rand(d, generator=gen, device="cuda")
    st["decay"] = torch.log(torch.expm1(-torch.log(keep) / _SCALE))
    b = case["batch"]
    rows = (b, d) if case["op"] == "rec_step" else (b, case["length"], d)
    st.update(x=normal(*rows), decay_gate=normal(*rows), input_gate=normal(*rows))
    st["state"] = torch.randn((b, d), generator=gen, device="cuda")
    if case["op"] in ("rec_train", "rec_grad"):
        st["grad"] = normal(*rows, scale=1e-3)
    st["seq_idx"] = None
    if case.get("seqs", 1) > 1:
        ends = torch.rand((b, case["length"]), generator=gen, device="cuda") < case["seqs"] / case["length"]
        st["seq_idx"] = torch.cumsum(ends, 1).to(torch.int32)
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
    if op == "ff":
        return m.gated_feed_forward(st["x"], st["w_gate"], st["w_up"], st["w_down"], activation=case["act"])
    if op == "ff_grad":
        return m.gated_feed_forward_grad(st["x"], st["w_gate"], st["w_up"], st["w_down"], st["grad"], activation=case["act"])
    args = (st["x"], st["decay_gate"], st["input_gate"], st["decay"])
    if op == "rec_step":
        state, y = m.gated_recurrence_update(st["state"], *args, scale=_SCALE)
        return y, state
    kw = dict(scale=_SCALE, initial_state=st["state"], seq_idx=st["seq_idx"])
    if op == "rec":
        return m.gated_recurrence(*args, return_final_state=True, **kw)
    if op == "rec_grad":
        return m.gated_recurrence_grad(*args, st["grad"], **kw)
    y, final, checkpoints = m.gated_recurrence(*args, return_final_state=True, return_checkpoints=True, **kw)
    return (y, final) + tuple(m.gated_recurrence_grad(*args, st["grad"], checkpoints=checkpoints, **kw))


def _act(g, name):
    """An activation and its derivative."""
    if name == "relu":
        on = (g > 0).float()
        return g * on, on
    if name == "silu":
        s = 1 / (1 + torch.exp(-g))
        return g * s, s * (1 + g * (1 - s))
    if name == "gelu":
        p = 0.5 * (1 + torch.erf(g * math.sqrt(0.5)))
        return g * p, p + g * torch.exp(-0.5 * g * g) * (1 / math.sqrt(2 * math.pi))
    c = math.sqrt(2 / math.pi)
    t = torch.tanh(c * (g + 0.044715 * g * g * g))
    return 0.5 * g * (1 + t), 0.5 * (1 + t) + 0.5 * g * (1 - t * t) * c * (1 + 3 * 0.044715 * g * g)


def _scan(a, b):
    """h_t = a_t h_{t-1} + b_t along dim 1 by doubling: after step s each value holds the last 2 s terms."""
    s, n = 1, a.shape[1]
    while s < n:
        b = torch.cat([b[:, :s], b[:, s:] + a[:, s:] * b[:, :-s]], 1)
        a = torch.cat([a[:, :s], a[:, s:] * a[:, :-s]], 1)
        s *= 2
    return b


def run(st):
    if own:
        return _run_own(st)
    case = st["case"]
    op, dt = case["op"], _DT[case["dtype"]]
    x = st["x"].float()
    if op in ("ff", "ff_grad"):
        wg, wu, wd = st["w_gate"].float(), st["w_up"].float(), st["w_down"].float()
        g, u = x @ wg.t(), x @ wu.t()
        v, dv = _act(g, case["act"])
        if op == "ff":
            return ((v * u) @ wd.t()).to(dt)
        dy = st["grad"].float()
        dh = dy @ wd
        dg, du = dh * u * dv, dh * v
        return (dg @ wg + du @ wu).to(dt), (dg.t() @ x).to(dt), (du.t() @ x).to(dt), (dy.t() @ (v * u)).to(dt)
    r, i, lam, state = st["decay_gate"].float(), st["input_gate"].float(), st["decay"], st["state"]
    softplus = torch.log1p(torch.exp(lam))
    s_r, s_i = 1 / (1 + torch.exp(-r)), 1 / (1 + torch.exp(-i))
    la = -_SCALE * softplus * s_r
    a = 1 + torch.expm1(la)  # as near to 1 as float32 goes: over thousands of steps its error is what counts
    beta = torch.sqrt(-torch.expm1(2 * la))
    if op == "rec_step":
        h = a * state + beta * s_i * x
        return h.to(dt), h
    # what is left of the state before: nothing where a packed sequence starts
    c = a
    if st["seq_idx"] is not None:
        starts = st["seq_idx"][:, 1:] != st["seq_idx"][:, :-1]
        c = torch.cat([a[:, :1], torch.where(starts[:, :, None], torch.zeros_like(a[:, 1:]), a[:, 1:])], 1)
    b = beta * s_i * x
    h = _scan(c, torch.cat([b[:, :1] + (c[:, 0] * state)[:, None], b[:, 1:]], 1))
    if op == "rec":
        return h.to(dt), h[:, -1]
    before = torch.cat([state[:, None], h[:, :-1]], 1)
    after = torch.cat([c[:, 1:], torch.zeros_like(c[:, :1])], 1)
    delta = _scan(after.flip(1), st["grad"].float().flip(1)).flip(1)
    q = torch.where(beta > 0, la / beta, torch.zeros_like(la))
    m = delta * (c * la * before - a * a * q * s_i * x)
    dx = delta * beta * s_i
    grads = (dx.to(dt), (m * (1 - s_r)).to(dt), (dx * x * (1 - s_i)).to(dt),
             m.sum((0, 1)) / ((1 + torch.exp(-lam)) * softplus), c[:, 0] * delta[:, 0])
    return grads if op == "rec_grad" else (h.to(dt), h[:, -1]) + grads


def work(case):
    es = 4 if case["dtype"] == "f32" else 2
    d = case["d"]
    if case["op"].startswith("ff"):
        t, f = case["tokens"], case["f"]
        if case["op"] == "ff":
            return {"bytes": (2 * t * d + 3 * d * f) * es, "flops": 6 * t * d * f}
        return {"bytes": (3 * t * d + 6 * d * f) * es, "flops": 16 * t * d * f}
    n = case["batch"] * d
    if case["op"] == "rec_step":
        return {"bytes": n * (4 * es + 8) + 4 * d, "flops": 20 * n}
    values = n * case["length"]
    extra = 8 * n + 4 * d + (4 * case["batch"] * case["length"] if case["seqs"] > 1 else 0)
    tensors, ops = {"rec": (4, 20), "rec_grad": (7, 45), "rec_train": (8, 65)}[case["op"]]
    return {"bytes": values * tensors * es + extra, "flops": values * ops}


def exact(case, seed):
    st = prepare(case, seed)
    f64 = torch.float64
    if case["op"].startswith("ff"):
        leaves = [st[n].to(f64).requires_grad_(case["op"] == "ff_grad") for n in ("x", "w_gate", "w_up", "w_down")]
        x, wg, wu, wd = leaves
        fn = {"relu": torch.relu, "silu": torch.nn.functional.silu, "gelu": torch.nn.functional.gelu,
              "gelu_tanh": lambda v: torch.nn.functional.gelu(v, approximate="tanh")}[case["act"]]
        y = (fn(x @ wg.T) * (x @ wu.T)) @ wd.T
        return y if case["op"] == "ff" else torch.autograd.grad(y, leaves, st["grad"].to(f64))
    x, r, i, lam = (st[n].to(f64) for n in ("x", "decay_gate", "input_gate", "decay"))
    state = st["state"].to(f64)
    k = _SCALE * torch.nn.functional.softplus(lam)
    open_r, open_i = torch.sigmoid(r), torch.sigmoid(i)
    la = k.neg() * open_r
    a, a2 = la.exp(), (2 * la).exp()
    root = torch.expm1(2 * la).neg().sqrt()
    fed = root * open_i * x
    if case["op"] == "rec_step":
        h = a * state + fed
        return h, h
    n = case["length"]
    if st["seq_idx"] is not None:
        kept = torch.ones(x.shape[:2], dtype=f64, device="cuda")
        kept[:, 1:] = (st["seq_idx"][:, 1:] == st["seq_idx"][:, :-1]).to(f64)
        a = a * kept[:, :, None]
    h = torch.empty_like(fed)
    last = state
    for t in range(n):
        last = torch.addcmul(fed[:, t], a[:, t], last, out=h[:, t])
    if case["op"] == "rec":
        return h, h[:, -1]
    delta = st["grad"].to(f64)
    for t in range(n - 2, -1, -1):
        delta[:, t].addcmul_(a[:, t + 1], delta[:, t + 1])
    # d root / d la = -a^2 / root
    dla = delta * (torch.cat([state[:, None], h[:, :-1]], 1) * a - a2 / root * open_i * x)
    grads = (delta * root * open_i, dla * la * (1 - open_r), delta * root * x * open_i * (1 - open_i),
             -(dla * open_r).sum((0, 1)) * _SCALE * torch.sigmoid(lam), a[:, 0] * delta[:, 0])
    return grads if case["op"] == "rec_grad" else (h, h[:, -1]) + grads
