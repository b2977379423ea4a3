"""Token embedding and its gradient, linear cross entropy and its gradients, gradient clipping:
the CUDA kernels against plain float64 restatements, and their refusals.

Tolerances.  u = 2^-24 is the unit roundoff of float32 and v = 2^-8 of bfloat16 (8 significant bits).
- lookup: one float32 product, rounded once to the output type: equal bits.
- embedding gradient: a sum of n terms in float32, times the scale: |error| <= (n + 2) u sum|g| |scale|,
  plus v |result| where the output is bfloat16.
- loss, bfloat16 inputs: products are exact in float32 and D of them are added on the tensor
  cores, whose adds may truncate (2u): a logit is off by at most 2 D u sum|x w|, the loss by twice
  the largest of a row, plus 4 u (1 + |loss|) for the exponentials' and logarithm's own rounding.
- loss, float32 inputs: two bfloat16 terms per value leave v^2 = 2^-16 of it, and lo * lo, below 2^-16
  of the product, is dropped: 3 * 2^-16 sum|x w| is added to a logit's error.
- gradients: relative 2-norm.  bfloat16: dl is rounded once (v), the result once (v), and the logits'
  error enters as an absolute error of log dl: 2 v + 2 * max logit error + 1e-4.  float32: three
  products leave 3 * 2^-16, dl's own two terms 2^-16, again the logits' error, and the adds.
- clipping: the factor is correct to u, the product to u (v for bfloat16).
"""
import math

import numpy as np
import pytest
import torch

from mamba2_b200 import (clip_grad_norm, embedding, embedding_grad, grad_norm, linear_cross_entropy,
                         linear_cross_entropy_grad)

gpu = pytest.mark.gpu
U, V = 2.0 ** -24, 2.0 ** -8
DT = {"f32": torch.float32, "bf16": torch.bfloat16}


@pytest.fixture(autouse=True)
def _need_gpu(request):
    if request.node.get_closest_marker("gpu") and not torch.cuda.is_available():
        pytest.skip("no CUDA device")


def rnd(*shape, dtype="f32", seed=0, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * scale).to(DT[dtype])


def f64(t):
    return t.detach().double().cpu()


def same_bits(a, b):
    return torch.equal(a.cpu().reshape(-1).view(torch.uint8), b.cpu().reshape(-1).view(torch.uint8))


# ---------------------------------------------------------------------------------------------
# embedding
# ---------------------------------------------------------------------------------------------
def ids_for(kind, n, vocab, seed=1):
    g = torch.Generator().manual_seed(seed)
    if kind == "one":
        return torch.full((n,), vocab - 1, dtype=torch.int64)
    if kind == "zipf":
        return (torch.exp(torch.rand(n, generator=g) * math.log(vocab)) - 1).long().clamp(0, vocab - 1)
    if kind == "sorted":
        return torch.arange(n) % vocab
    return torch.randint(0, vocab, (n,), generator=g)


@gpu
@pytest.mark.parametrize("n,vocab,dim", [(1, 1, 1), (1, 50257, 768), (7, 11, 8), (33, 100, 257), (256, 1000, 2560),
                                         (1000, 37, 1031), (3, 5, 8200)])
@pytest.mark.parametrize("wd,od", [("bf16", "bf16"), ("bf16", "f32"), ("f32", "f32"), ("f32", "bf16")])
def test_embedding_bits(n, vocab, dim, wd, od):
    w = rnd(vocab, dim, dtype=wd)
    ids = ids_for("uniform", n, vocab)
    scale = math.sqrt(dim)
    out = embedding(ids.cuda(), w.cuda(), scale=scale, out_dtype=DT[od])
    ref = (w[ids].float() * np.float32(scale)).to(DT[od])
    assert out.dtype == DT[od] and same_bits(out, ref)


@gpu
@pytest.mark.parametrize("idt", [torch.int32, torch.int64])
def test_embedding_drops_and_strides(idt):
    base = rnd(50, 3, 64, dtype="bf16").cuda()
    w = base[:, 1]                                  # rows 192 apart, start not at the buffer's
    odd = rnd(50, 67, dtype="bf16").cuda()[:, 3:]   # rows 67 apart, not 16-byte aligned
    ids = torch.tensor([[0, 49, -1, 50], [7, 2 ** 31 - 1, -2 ** 31, 3]], dtype=idt).cuda()
    keep = ((ids >= 0) & (ids < 50) & (ids != 7)).cpu()
    for t in (w, odd):
        out = embedding(ids, t, padding_idx=7)
        ref = torch.where(keep[..., None], t.cpu()[ids.long().clamp(0, 49).cpu()], torch.zeros((), dtype=t.dtype))
        assert out.shape == (2, 4, 64) and same_bits(out, ref)
    # transposed ids, no ids
    assert same_bits(embedding(ids.t(), w), embedding(ids.t().contiguous(), w))
    assert embedding(ids[:0], w).shape == (0, 4, 64)


@gpu
def test_embedding_keeps_infinities_and_nan():
    w = torch.tensor([[float("inf")] * 8, [float("nan")] * 8, [-0.0] * 8])
    out = embedding(torch.tensor([0, 1, 2, 5]).cuda(), w.cuda(), scale=2.0).cpu()
    assert torch.isinf(out[0]).all() and torch.isnan(out[1]).all() and torch.signbit(out[2]).all()
    assert (out[3] == 0).all()


def ref_embedding_grad(ids, g, vocab, scale, pad=None):
    """(sums, sum of magnitudes, terms) per row in float64."""
    keep = (ids >= 0) & (ids < vocab)
    if pad is not None:
        keep &= ids != pad
    s = torch.zeros(vocab, g.shape[1], dtype=torch.float64)
    a = torch.zeros_like(s)
    s.index_add_(0, ids[keep], f64(g)[keep])
    a.index_add_(0, ids[keep], f64(g)[keep].abs())
    n = torch.bincount(ids[keep], minlength=vocab).double()[:, None]
    return s * scale, a * abs(scale), n


@gpu
@pytest.mark.parametrize("kind", ["uniform", "zipf", "one", "sorted"])
@pytest.mark.parametrize("n,vocab,dim", [(1, 1, 1), (1, 600, 8), (31, 7, 264), (32, 513, 100), (65, 3, 16),
                                         (777, 512, 768), (5000, 70000, 40), (9000, 300, 257)])
@pytest.mark.parametrize("gd,od", [("bf16", "bf16"), ("f32", "f32"), ("bf16", "f32"), ("f32", "bf16")])
def test_embedding_grad(kind, n, vocab, dim, gd, od):
    ids, g = ids_for(kind, n, vocab), rnd(n, dim, dtype=gd, seed=2)
    out = embedding_grad(ids.cuda(), g.cuda(), vocab, scale=0.37, out_dtype=DT[od])
    s, a, cnt = ref_embedding_grad(ids, g, vocab, float(np.float32(0.37)))
    bound = (cnt + 2) * U * a + (V * s.abs() if od == "bf16" else 0)
    assert out.shape == (vocab, dim) and out.dtype == DT[od]
    err = (f64(out) - s).abs()
    assert (err <= bound).all(), float((err - bound).max())


@gpu
@pytest.mark.parametrize("vocab", [1, 2, 511, 512, 513, 1 << 18, (1 << 18) + 1])
def test_embedding_grad_radix_edges(vocab):
    """Vocabularies at the digits' borders (the largest key is vocab itself, for what is dropped)."""
    g = torch.Generator().manual_seed(5)
    ids = torch.randint(-1, vocab + 1, (3000,), generator=g)
    ids[:4] = torch.tensor([vocab - 1, 0, vocab, -5])
    x = rnd(3000, 8, seed=6)
    out = embedding_grad(ids.cuda(), x.cuda(), vocab)
    s, a, cnt = ref_embedding_grad(ids, x, vocab, 1.0)
    assert ((f64(out) - s).abs() <= (cnt + 2) * U * a).all()


@gpu
@pytest.mark.parametrize("n,vocab", [(5001, v) for v in (1, 2, 511, 512, 513, 1 << 18, (1 << 18) + 1)] +
                         [(4096, 777), (4097, 777), (4096, (1 << 20) - 1), (4096, 1 << 20), (129, 5), (128, 1), (1, 3)])
def test_embedding_grad_both_sorts(n, vocab):
    """Few ids are placed by counting, more by digits: sizes on both sides of the change."""
    g = torch.Generator().manual_seed(n)
    ids = torch.randint(-1, vocab + 1, (n,), generator=g)
    ids[0] = vocab - 1
    x = rnd(n, 4, seed=8)
    for t in (ids, ids.int()):
        out = embedding_grad(t.cuda(), x.cuda(), vocab)
        s, a, cnt = ref_embedding_grad(ids, x, vocab, 1.0)
        assert ((f64(out) - s).abs() <= (cnt + 2) * U * a).all()


@gpu
@pytest.mark.parametrize("vocab,dim,od", [(1 << 19, 130, "f32"), (100001, 1367, "bf16"), (3000, 1, "bf16"), (3000, 7, "bf16"),
                                          (3000, 9, "f32"), (3000, 33, "bf16"), (3000, 127, "f32")])
def test_embedding_grad_zero_rows(vocab, dim, od):
    """Every other row is written with zeros: wide and narrow rows, aligned or not, large tables."""
    ids, x = ids_for("uniform", 300, vocab), rnd(300, dim, dtype=od, seed=9)
    ic, xc = ids.cuda(), x.cuda()
    torch.full((vocab, dim), float("nan"), device="cuda", dtype=DT[od])   # what the allocator hands out next
    out = embedding_grad(ic, xc, vocab)
    named = torch.zeros(vocab, dtype=torch.bool, device="cuda")
    named[ic] = True
    assert not out[~named].any() and not torch.isnan(out[~named]).any()
    s, a, cnt = ref_embedding_grad(ids, x, vocab, 1.0)
    bound = (cnt + 2) * U * a + (V * s.abs() if od == "bf16" else 0)
    rows = ids.unique()
    assert ((f64(out[rows.cuda()]) - s[rows]).abs() <= bound[rows]).all()


@gpu
def test_embedding_grad_large_sort_and_repeatable():
    """Several tokens per sorting lane, runs over many pieces; equal bits in every run."""
    ids, g = ids_for("zipf", 200001, 50000), rnd(200001, 24, dtype="bf16", seed=3)
    ic, gc = ids.cuda(), g.cuda()
    out = embedding_grad(ic, gc, 50000, out_dtype=torch.float32)
    s, a, cnt = ref_embedding_grad(ids, g, 50000, 1.0)
    assert ((f64(out) - s).abs() <= (cnt + 2) * U * a).all()
    for _ in range(3):
        assert same_bits(out, embedding_grad(ic, gc, 50000, out_dtype=torch.float32))


@gpu
@pytest.mark.parametrize("od", ["f32", "bf16"])
def test_embedding_grad_accumulates_and_drops(od):
    vocab, dim = 100, 48
    ids = torch.tensor([[3, 3, -1], [99, 100, 7], [7, 5, 3]])
    wide = rnd(3, 3, 60, seed=4).cuda()
    g = wide[..., 5:53]                                  # rows 60 apart, unaligned start
    old = rnd(vocab, 64, dtype=od, seed=5).cuda()
    acc = old.clone()[:, 8:56]
    before = acc.clone()
    ret = embedding_grad(ids.cuda(), g, vocab, scale=2.0, padding_idx=5, accumulate_into=acc)
    assert ret is acc
    s, a, cnt = ref_embedding_grad(ids.reshape(-1), g.cpu().reshape(-1, dim), vocab, 2.0, pad=5)
    ref = f64(before) + s
    bound = (cnt + 3) * U * (a + f64(before).abs()) + (V * ref.abs() if od == "bf16" else 0)
    bound[cnt[:, 0] == 0] = 0                            # rows that no token names keep their bits
    assert ((f64(acc) - ref).abs() <= bound).all()
    # nothing to add; and a dense gradient of nothing is zero
    assert same_bits(embedding_grad(ids[:0].cuda(), g[:0], vocab, accumulate_into=acc.clone()), acc)
    z = embedding_grad(ids[:0].cuda(), g[:0], vocab)
    assert z.shape == (vocab, dim) and (z == 0).all()
    z = embedding_grad(torch.full((40,), -1).cuda(), torch.full((40, dim), float("nan")).cuda(), vocab)
    assert (z == 0).all()


@gpu
def test_embedding_grad_is_the_gradient_by_differences():
    """sum(embedding(W) * g) is linear in W: its difference along any direction is <dW, direction>."""
    vocab, dim, n = 40, 24, 100
    w, d = rnd(vocab, dim, seed=1).double(), rnd(vocab, dim, seed=2).double()
    g, ids = rnd(n, dim, seed=3), ids_for("zipf", n, vocab)
    f = lambda m: float((m[ids] * 1.5 * g.double()).sum())
    dw = embedding_grad(ids.cuda(), g.cuda(), vocab, scale=1.5)
    num = (f(w + 0.5 * d) - f(w - 0.5 * d))
    assert abs(num - float((f64(dw) * d).sum())) <= 1e-4 * float((f64(dw) * d).abs().sum())


# ---------------------------------------------------------------------------------------------
# linear cross entropy
# ---------------------------------------------------------------------------------------------
def ref_ce(x, w, y, ignore=-100, reduction="mean", grad_loss=None):
    x, w = f64(x).reshape(-1, x.shape[-1]), f64(w)
    y = y.reshape(-1).cpu()
    s = x @ w.t()
    mag = x.abs() @ w.abs().t()
    lse = torch.logsumexp(s, 1)
    counted = y != ignore
    col = torch.where(counted, y, torch.zeros_like(y))
    loss = torch.where(counted, lse - s.gather(1, col[:, None])[:, 0], torch.zeros_like(lse))
    c = counted.double()
    if reduction == "none":
        c = c if grad_loss is None else c * f64(grad_loss).reshape(-1)
        total = loss
    else:
        k = max(1, int(counted.sum())) if reduction == "mean" else 1
        c = c / k * (1.0 if grad_loss is None else float(grad_loss))
        total = loss.sum() / k
    dl = torch.exp(s - lse[:, None])
    dl[torch.arange(len(y)), col] -= 1.0
    dl *= c[:, None]
    return dict(loss=total, rows=loss, lse=lse, dx=dl @ w, dw=dl.t() @ x, mag=mag.max(1).values)


def logit_error(r, dim, dtype):
    e = 2 * dim * U * r["mag"]
    return e if dtype == "bf16" else e + 3 * 2.0 ** -16 * r["mag"]


def rel(got, ref):
    d = float(ref.norm())
    return float((f64(got).reshape(ref.shape) - ref).norm()) / (d if d else 1.0)


def ce_inputs(t, v, d, dtype, seed=0, ignored=0.0, ignore=-100, gain=6.0):
    g = torch.Generator().manual_seed(seed)
    w = rnd(v, d, dtype=dtype, seed=seed + 1, scale=1 / math.sqrt(d))
    y = torch.randint(0, v, (t,), generator=g)
    x = (rnd(t, d, seed=seed + 2) + gain * torch.rand(t, 1, generator=g) * w[y].float()).to(DT[dtype])
    if ignored:
        y = torch.where(torch.rand(t, generator=g) < ignored, torch.full_like(y, ignore), y)
    return x, w, y


def grad_bound(r, dim, dtype):
    e = float(logit_error(r, dim, dtype).max())
    # 1e-4 and 1e-5: the adds of the gradients' own products, up to a few thousand of them
    return 2 * V + 2 * e + 1e-4 if dtype == "bf16" else 4 * 2.0 ** -16 + 2 * e + 1e-5


SIZES = [(1, 1, 1), (1, 2, 8), (1, 3001, 64), (3, 255, 72), (7, 257, 100), (64, 513, 65), (127, 1000, 40),
         (128, 256, 64), (129, 2049, 128), (200, 1023, 200), (257, 4096, 264), (300, 131, 1000),
         # the forms for a few tokens: every row width, widths past one column block, past one pass
         (2, 500, 96), (2, 37, 1025), (4, 777, 260), (4, 9, 2056), (5, 60, 1031), (8, 3000, 72), (8, 300, 33),
         (9, 400, 128), (20, 300, 64), (32, 700, 48), (33, 700, 48)]


@gpu
@pytest.mark.parametrize("t,v,d", SIZES)
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_linear_cross_entropy_rows(t, v, d, dtype):
    x, w, y = ce_inputs(t, v, d, dtype)
    loss, lse = linear_cross_entropy(x.cuda(), w.cuda(), y.cuda(), reduction="none", return_lse=True, check_status=True)
    r = ref_ce(x, w, y, reduction="none")
    bound = 2 * logit_error(r, d, dtype) + 4 * U * (1 + r["rows"].abs() + r["lse"].abs())
    assert loss.dtype == torch.float32 and loss.shape == (t,)
    assert ((f64(loss) - r["rows"]).abs() <= bound).all()
    assert ((f64(lse) - r["lse"]).abs() <= bound).all()


@gpu
@pytest.mark.parametrize("t,v,d", SIZES)
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("reduction", ["mean", "none"])
def test_linear_cross_entropy_grads(t, v, d, dtype, reduction):
    x, w, y = ce_inputs(t, v, d, dtype, seed=3, ignored=0.3 if t > 4 else 0.0)
    gl = rnd(t, seed=9) if reduction == "none" else torch.tensor(3.0)
    loss, dx, dw = linear_cross_entropy_grad(x.cuda(), w.cuda(), y.int().cuda(), reduction=reduction,
                                             grad_loss=gl.cuda(), check_status=True)
    r = ref_ce(x, w, y, reduction=reduction, grad_loss=gl)
    assert dx.dtype == DT[dtype] and dw.dtype == DT[dtype] and dx.shape == (t, d) and dw.shape == (v, d)
    tol = grad_bound(r, d, dtype)
    # a vocabulary of one word: the gradients are zero, up to the logits' rounding
    if v == 1:
        assert float(f64(dx).abs().max()) <= 1e-5 and float(f64(dw).abs().max()) <= 1e-5
    else:
        assert rel(dx, r["dx"]) <= tol, rel(dx, r["dx"])
        assert rel(dw, r["dw"]) <= tol, rel(dw, r["dw"])
    # the same loss as the call without gradients
    other = linear_cross_entropy(x.cuda(), w.cuda(), y.cuda(), reduction=reduction)
    assert torch.allclose(loss, other, rtol=1e-6, atol=1e-6)


@gpu
def test_linear_cross_entropy_partial_outputs():
    x, w, y = ce_inputs(150, 700, 96, "bf16")
    args = (x.cuda(), w.cuda(), y.cuda())
    loss, dx, dw = linear_cross_entropy_grad(*args, weight_grad_dtype=torch.float32)
    l1, dx1, none = linear_cross_entropy_grad(*args, need_weight_grad=False)
    l2, none2, dw2 = linear_cross_entropy_grad(*args, need_hidden_grad=False, weight_grad_dtype=torch.float32)
    assert none is None and none2 is None and dw.dtype == torch.float32
    assert same_bits(dx, dx1) and same_bits(dw, dw2) and same_bits(loss, l1) and same_bits(loss, l2)
    assert rel(dw, ref_ce(x, w, y)["dw"]) <= V + 1e-4 + 2 * float(logit_error(ref_ce(x, w, y), 96, "bf16").max())
    # equal calls, equal bits
    again = linear_cross_entropy_grad(*args, weight_grad_dtype=torch.float32)
    assert all(same_bits(a, b) for a, b in zip((loss, dx, dw), again))


@gpu
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_linear_cross_entropy_strides_and_shapes(dtype):
    x, w, y = ce_inputs(60, 333, 88, dtype, ignored=0.2)
    r = ref_ce(x, w, y)
    wide_x = torch.full((60, 99), float("nan"), dtype=DT[dtype]).cuda()
    wide_w = torch.full((333, 96), float("nan"), dtype=DT[dtype]).cuda()
    wide_x[:, 3:91] = x.cuda()        # unaligned rows
    wide_w[:, :88] = w.cuda()         # aligned rows, further apart than they are long
    yt = y.cuda().reshape(5, 12).t().contiguous().t()   # targets in another order of memory
    loss, dx, dw = linear_cross_entropy_grad(wide_x[:, 3:91].unflatten(0, (5, 12)), wide_w[:, :88], yt)
    assert dx.shape == (5, 12, 88) and abs(float(loss) - float(r["loss"])) <= 1e-4
    tol = grad_bound(r, 88, dtype)
    assert rel(dx, r["dx"]) <= tol and rel(dw, r["dw"]) <= tol


@gpu
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_linear_cross_entropy_nothing_counts(dtype):
    x, w, y = ce_inputs(130, 300, 64, dtype)
    none = torch.full_like(y, -7)
    for red in ("mean", "sum"):
        loss, dx, dw = linear_cross_entropy_grad(x.cuda(), w.cuda(), none.cuda(), ignore_index=-7, reduction=red)
        assert float(loss) == 0 and (dx == 0).all() and (dw == 0).all()
    rows = linear_cross_entropy(x.cuda(), w.cuda(), none.cuda(), ignore_index=-7, reduction="none")
    assert (rows == 0).all()
    # an ignore_index inside the vocabulary is ignored too
    y[:60] = 5
    r = ref_ce(x, w, y, ignore=5)
    loss, dx, _ = linear_cross_entropy_grad(x.cuda(), w.cuda(), y.cuda(), ignore_index=5)
    assert abs(float(loss) - float(r["loss"])) <= 1e-4 and (dx[:60] == 0).all()
    # no tokens at all
    loss, dx, dw = linear_cross_entropy_grad(x[:0].cuda(), w.cuda(), y[:0].cuda())
    assert float(loss) == 0 and dx.shape == (0, 64) and (dw == 0).all()


@gpu
def test_linear_cross_entropy_ignored_rows_may_hold_anything():
    """What an ignored position holds (padding, infinities, NaN) reaches neither loss nor gradients of
    the others; its own gradient is zero."""
    x, w, y = ce_inputs(140, 500, 64, "bf16")
    r = ref_ce(x[:100], w, y[:100])
    y[100:] = -100
    x[100:] = 0
    loss, dx, dw = linear_cross_entropy_grad(x.cuda(), w.cuda(), y.cuda())
    tol = grad_bound(r, 64, "bf16")
    assert abs(float(loss) - float(r["loss"])) <= 1e-4
    assert rel(dx[:100], r["dx"]) <= tol and rel(dw, r["dw"]) <= tol and (dx[100:] == 0).all()
    for bad in (float("inf"), float("nan"), torch.finfo(torch.bfloat16).min):
        x2 = x.clone()
        x2[100:] = bad
        l2, dx2, dw2 = linear_cross_entropy_grad(x2.cuda(), w.cuda(), y.cuda())
        assert same_bits(loss, l2) and same_bits(dx, dx2) and same_bits(dw, dw2)


@gpu
def test_linear_cross_entropy_invalid_targets_and_nonfinite_rows():
    x, w, y = ce_inputs(20, 90, 32, "f32")
    y[3], y[4] = 90, -1
    rows = linear_cross_entropy(x.cuda(), w.cuda(), y.cuda(), reduction="none").cpu()
    assert torch.isnan(rows[3]) and torch.isnan(rows[4]) and torch.isfinite(rows[torch.arange(20) > 4]).all()
    x2 = x.clone()
    x2[0] = float("nan")
    rows2 = linear_cross_entropy(x2.cuda(), w.cuda(), y.cuda(), reduction="none").cpu()
    assert torch.isnan(rows2[0]) and torch.equal(rows[5:], rows2[5:])


@gpu
@pytest.mark.parametrize("shift", [0.0, 300.0, -300.0])
def test_linear_cross_entropy_large_logits(shift):
    """Logits far from zero: the running maximum keeps the sums in range."""
    t, v, d = 40, 700, 64
    x, w, y = ce_inputs(t, v, d, "bf16", gain=0.0)
    x[:, 0] = 16.0
    w[:, 0] = shift / 16.0
    x = (x.float() * 3).bfloat16()
    loss = linear_cross_entropy(x.cuda(), w.cuda(), y.cuda(), reduction="none")
    r = ref_ce(x, w, y, reduction="none")
    bound = 2 * logit_error(r, d, "bf16") + 4 * U * (1 + r["lse"].abs())
    assert ((f64(loss) - r["rows"]).abs() <= bound).all()


@gpu
def test_linear_cross_entropy_confident_tokens():
    """p of the target near 1: the loss and p - 1 keep their relative accuracy."""
    d, v = 64, 400
    w = rnd(v, d, seed=1, scale=1 / 8)
    y = torch.arange(16)
    x = 60.0 * w[y] / (w[y] * w[y]).sum(1, keepdim=True) * 0.5
    loss, dx, _ = linear_cross_entropy_grad(x.cuda(), w.cuda(), y.cuda(), reduction="sum")
    r = ref_ce(x, w, y, reduction="sum")
    e = float(logit_error(r, d, "f32").max())
    assert float(r["loss"]) < 1e-3 * 16
    assert abs(float(loss) - float(r["loss"])) <= (2 * e + 1e-5) * float(r["loss"]) + 1e-9 + 16 * 2 * e * 1e-3
    assert rel(dx, r["dx"]) <= 4 * e + 4 * 2.0 ** -16 + 1e-5


@gpu
def test_linear_cross_entropy_grad_by_differences():
    """Directional differences of the float64 loss against the kernel's gradients."""
    x, w, y = ce_inputs(48, 300, 40, "f32", ignored=0.2)
    _, dx, dw = linear_cross_entropy_grad(x.cuda(), w.cuda(), y.cuda())
    ex, ew = rnd(48, 40, seed=20).double(), rnd(300, 40, seed=21).double()
    h = 1e-4
    f = lambda s: float(ref_ce(x.double() + s * h * ex, w.double() + s * h * ew, y)["loss"])
    num = (f(1) - f(-1)) / (2 * h)
    ana = float((f64(dx) * ex).sum() + (f64(dw) * ew).sum())
    size = float((f64(dx) * ex).norm() + (f64(dw) * ew).norm())
    assert abs(num - ana) <= 1e-4 * size + 1e-7


@gpu
def test_linear_cross_entropy_token_chunks():
    """More tokens than one chunk of the workspace holds (130000 logits a row): the weight's gradient
    is summed over the chunks; sampled rows against float64."""
    t, v, d = 4500, 131072, 64
    g = torch.Generator(device="cuda").manual_seed(0)
    w = (torch.randn(v, d, generator=g, device="cuda") / 8).bfloat16()
    y = torch.randint(0, v, (t,), generator=g, device="cuda")
    x = (torch.randn(t, d, generator=g, device="cuda") + 4 * w[y].float()).bfloat16()
    loss, dx, dw = linear_cross_entropy_grad(x, w, y, check_status=True)
    xs, ws = x.double(), w.double()
    total, dws = 0.0, torch.zeros_like(ws)
    dxs = torch.empty_like(xs)
    for lo in range(0, t, 500):
        s = xs[lo:lo + 500] @ ws.t()
        lse = torch.logsumexp(s, 1, keepdim=True)
        total += float((lse[:, 0] - s.gather(1, y[lo:lo + 500, None])[:, 0]).sum())
        p = torch.exp(s - lse)
        p[torch.arange(len(p)), y[lo:lo + 500]] -= 1
        dxs[lo:lo + 500] = p @ ws / t
        dws += p.t() @ xs[lo:lo + 500] / t
    assert abs(float(loss) - total / t) <= 1e-5 * total / t
    assert rel(dx, dxs.cpu()) <= 2 * V + 1e-3 and rel(dw, dws.cpu()) <= 2 * V + 1e-3


@gpu
def test_lm_ops_on_another_stream():
    x, w, y = ce_inputs(100, 500, 64, "bf16")
    xc, wc, yc = x.cuda(), w.cuda(), y.cuda()
    want = linear_cross_entropy_grad(xc, wc, yc)
    e_want = embedding_grad(yc, xc, 500)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        torch.cuda._sleep(2_000_000)
        got = linear_cross_entropy_grad(xc * 1, wc * 1, yc * 1)
        e_got = embedding_grad(yc * 1, xc * 1, 500)
        _, norm = clip_grad_norm([got[1], got[2]], 0.5)
    s.synchronize()
    assert all(same_bits(a, b) for a, b in zip(want, got)) and same_bits(e_want, e_got)
    assert abs(float(norm) - float(torch.cat([want[1].flatten(), want[2].flatten()]).double().norm())) < 1e-5


@gpu
def test_lm_ops_in_a_graph():
    """All calls can be captured: no synchronisation, no copies from the host."""
    x, w, y = (t.cuda() for t in ce_inputs(70, 300, 64, "bf16"))

    def step():
        h = embedding(y, w, scale=2.0)
        loss, dx, dw = linear_cross_entropy_grad(h, w, y)
        dw = embedding_grad(y, dx, 300, scale=2.0, accumulate_into=dw)
        (g,), norm = clip_grad_norm([dw], 0.01)
        return loss, g, norm

    want = step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    graph.replay()
    torch.cuda.synchronize()
    assert all(same_bits(a, b) for a, b in zip(want, got))


# ---------------------------------------------------------------------------------------------
# gradient norm and clipping
# ---------------------------------------------------------------------------------------------
def grad_list(sizes, dtypes, seed=0):
    return [rnd(*s, dtype=dtypes[i % len(dtypes)], seed=seed + i, scale=10.0 ** (i % 4 - 2)) for i, s in enumerate(sizes)]


def ref_norm(ts):
    return math.sqrt(sum(float((f64(t) ** 2).sum()) for t in ts))


CLIP_SIZES = [[(1,)], [(3,), (0,), (8192,), (8193,)], [(5, 7), (1,), (100000,), (33, 65)], [(2,)] * 70,
              [(i % 50 + 1,) for i in range(1203)]]


@gpu
@pytest.mark.parametrize("sizes", CLIP_SIZES, ids=["one", "edges", "mixed", "70", "1203"])
@pytest.mark.parametrize("dtypes", [("f32",), ("bf16",), ("f32", "bf16")], ids=["f32", "bf16", "mixed"])
@pytest.mark.parametrize("where", ["new", "inplace", "out"])
def test_clip_grad_norm(sizes, dtypes, where):
    ts = grad_list(sizes, dtypes)
    n = ref_norm(ts)
    for max_norm in (0.5 * n, 2.0 * n + 1.0):
        dev = [t.cuda() for t in ts]
        keep = [t.clone() for t in dev]
        assert abs(float(grad_norm(dev)) - n) <= 2 * U * n
        out = None
        if where == "out":   # pieces of one float32 buffer, at any alignment
            flat = torch.full((sum(t.numel() for t in ts) + 1,), 7.0).cuda()
            out, at = [], 1
            for t in ts:
                out.append(flat[at:at + t.numel()].view(t.shape))
                at += t.numel()
        got, norm = clip_grad_norm(dev, max_norm, out=out, inplace=where == "inplace")
        assert norm.shape == () and abs(float(norm) - n) <= 2 * U * n
        c = min(1.0, max_norm / (n + 1e-6))
        for g, t, k in zip(got, ts, keep):
            ref = f64(t) * c
            bound = (4 * U + (V if g.dtype == torch.bfloat16 else 0)) * ref.abs()
            assert g.shape == t.shape and ((f64(g) - ref).abs() <= bound).all()
            if c == 1.0 and g.dtype == t.dtype:
                assert same_bits(g, t)
        if where == "inplace":
            assert all(a is b for a, b in zip(got, dev))
        else:
            assert all(same_bits(a, b) for a, b in zip(dev, keep))
        if where == "out":
            assert float(flat[0]) == 7.0


@gpu
def test_clip_grad_norm_repeats_and_range():
    ts = [t.cuda() for t in grad_list([(300000,), (17,), (4000, 11)], ("f32",))]
    a, b = grad_norm(ts), grad_norm(ts)
    assert same_bits(a, b)
    # squares outside the range of float32
    for s in (1e-30, 1e25):
        x = [torch.full((1000,), s).cuda(), torch.full((10,), -s).cuda()]
        n = math.sqrt(1010) * float(np.float32(s))
        assert abs(float(grad_norm(x)) - n) <= 4 * U * n
        got, _ = clip_grad_norm(x, 1.0)
        want = float(np.float32(s)) * min(1.0, 1.0 / (n + 1e-6))
        assert abs(float(got[1][0]) + want) <= 4 * U * want


@gpu
def test_clip_grad_norm_nonfinite_zero_and_strides():
    z = [torch.zeros(5).cuda(), torch.zeros(0, 3).cuda()]
    got, n = clip_grad_norm(z, 1.0)
    assert float(n) == 0 and (got[0] == 0).all() and got[1].shape == (0, 3)
    got, n = clip_grad_norm([torch.empty(0).cuda()], 1.0)
    assert float(n) == 0
    got, n = clip_grad_norm([torch.tensor([1.0, float("nan")]).cuda(), torch.ones(9).cuda()], 1.0)
    assert torch.isnan(n) and all(torch.isnan(g).all() for g in got)
    got, n = clip_grad_norm([torch.tensor([1.0, float("inf")]).cuda()], 1.0)
    assert torch.isinf(n) and float(got[0][0]) == 0 and torch.isnan(got[0][1])
    got, n = clip_grad_norm([torch.ones(4).cuda()], 0.0)
    assert float(n) == 2 and (got[0] == 0).all()
    t = rnd(30, 40, seed=3).cuda().t()
    got, n = clip_grad_norm([t], 1.0)
    assert abs(float(n) - ref_norm([t])) <= 2 * U * float(n)
    assert torch.allclose(f64(got[0]), f64(t) / float(n), rtol=1e-5)


# ---------------------------------------------------------------------------------------------
# offsets past 32 bits
# ---------------------------------------------------------------------------------------------
BIG_V, BIG_D = 540_001, 4096          # 2.2e9 values


@gpu
def test_offsets_past_32_bits_embedding():
    gen = torch.Generator(device="cuda").manual_seed(0)
    w = torch.empty((BIG_V, BIG_D), dtype=torch.bfloat16, device="cuda")
    w[-300:] = torch.randn((300, BIG_D), generator=gen, device="cuda").bfloat16()
    w[:300] = 1.0
    ids = torch.cat([torch.arange(BIG_V - 300, BIG_V), torch.arange(300)]).cuda()
    out = embedding(ids, w, scale=1.5)
    assert same_bits(out, (w[ids].float() * 1.5).bfloat16())
    g = torch.randn((600, BIG_D), generator=gen, device="cuda").bfloat16()
    dw = embedding_grad(ids, g, BIG_V)
    assert same_bits(dw[ids], g) and not bool(dw[300:-300].any())


@gpu
@pytest.mark.parametrize("t", [3, 40])
def test_offsets_past_32_bits_linear_cross_entropy(t):
    gen = torch.Generator(device="cuda").manual_seed(1)
    w = torch.randn((BIG_V, BIG_D), generator=gen, device="cuda", dtype=torch.bfloat16) / 64
    y = torch.randint(0, BIG_V, (t,), generator=gen, device="cuda")
    y[0], y[-1] = BIG_V - 1, 0
    x = (torch.randn((t, BIG_D), generator=gen, device="cuda") + 8 * w[y].float()).bfloat16()
    loss, dx, dw = linear_cross_entropy_grad(x, w, y, reduction="sum", check_status=True)
    # float64, in pieces of the vocabulary
    xs = x.double()
    lse = torch.full((t,), -float("inf"), dtype=torch.float64, device="cuda")
    for lo in range(0, BIG_V, 60000):
        lse = torch.logaddexp(lse, torch.logsumexp(xs @ w[lo:lo + 60000].double().t(), 1))
    rows = lse - (xs * w[y].double()).sum(1)
    assert abs(float(loss) - float(rows.sum())) <= 1e-5 * float(rows.sum())
    dxs = torch.zeros_like(xs)
    err = norm = 0.0
    for lo in range(0, BIG_V, 60000):
        p = torch.exp(xs @ w[lo:lo + 60000].double().t() - lse[:, None])
        for i, v in enumerate(y.tolist()):
            if lo <= v < lo + 60000:
                p[i, v - lo] -= 1.0
        dxs += p @ w[lo:lo + 60000].double()
        ref = p.t() @ xs
        err += float((dw[lo:lo + 60000].double() - ref).norm() ** 2)
        norm += float(ref.norm() ** 2)
    assert rel(dx, dxs.cpu()) <= 2 * V + 1e-3 and math.sqrt(err / norm) <= 2 * V + 1e-3


@gpu
def test_offsets_past_32_bits_clip():
    n = 2 ** 31 + 4099
    g = torch.ones(n, dtype=torch.bfloat16, device="cuda")
    g[-5:] = 3.0
    got, norm = clip_grad_norm([g], 1.0, inplace=True)
    want = math.sqrt(n - 5 + 45)
    assert abs(float(norm) - want) <= 2 * U * want
    c = 1.0 / (want + 1e-6)
    assert abs(float(got[0][-1]) - 3 * c) <= V * 3 * c and abs(float(got[0][2 ** 31]) - c) <= V * c
    assert abs(float(got[0][0]) - c) <= V * c


# ---------------------------------------------------------------------------------------------
# refusals (no GPU needed unless a CUDA tensor is)
# ---------------------------------------------------------------------------------------------
def test_refuse_cpu_tensors():
    ids, w, x = torch.zeros(3, dtype=torch.int64), torch.zeros(5, 8), torch.zeros(3, 8)
    for call in (lambda: embedding(ids, w), lambda: embedding_grad(ids, x, 5),
                 lambda: linear_cross_entropy(x, w, ids), lambda: linear_cross_entropy_grad(x, w, ids),
                 lambda: grad_norm([w]), lambda: clip_grad_norm([w], 1.0)):
        with pytest.raises(ValueError, match="CUDA"):
            call()


@gpu
def test_refusals():
    ids, w, x = torch.zeros(3, dtype=torch.int64).cuda(), torch.zeros(5, 8).cuda(), torch.zeros(3, 8).cuda()
    bad = [
        (TypeError, lambda: embedding(ids.float(), w)),
        (ValueError, lambda: embedding(ids, w[0])),
        (TypeError, lambda: embedding(ids, w.half())),
        (ValueError, lambda: embedding(ids, w, out_dtype=torch.float16)),
        (ValueError, lambda: embedding(ids, w, padding_idx=5)),
        (ValueError, lambda: embedding(ids, w[:0])),
        (ValueError, lambda: embedding_grad(ids, x[:2], 5)),
        (ValueError, lambda: embedding_grad(ids, x, 0)),
        (ValueError, lambda: embedding_grad(ids, x, 5, accumulate_into=w[:4])),
        (ValueError, lambda: embedding_grad(ids, x, 5, accumulate_into=torch.zeros(8, 5).cuda().t())),
        (TypeError, lambda: linear_cross_entropy(x, w, ids.short())),
        (TypeError, lambda: linear_cross_entropy(x.bfloat16(), w, ids)),
        (TypeError, lambda: linear_cross_entropy(x.half(), w.half(), ids)),
        (ValueError, lambda: linear_cross_entropy(x, w[:, :7], ids)),
        (ValueError, lambda: linear_cross_entropy(x, w, ids[:2])),
        (ValueError, lambda: linear_cross_entropy(x, w, ids, reduction="average")),
        (ValueError, lambda: linear_cross_entropy_grad(x, w, ids, grad_loss=torch.ones(3).cuda())),
        (ValueError, lambda: linear_cross_entropy_grad(x, w, ids, reduction="none", grad_loss=torch.ones(()).cuda())),
        (ValueError, lambda: linear_cross_entropy_grad(x, w, ids, weight_grad_dtype=torch.float16)),
        (ValueError, lambda: grad_norm([])),
        (TypeError, lambda: grad_norm([w.half()])),
        (TypeError, lambda: grad_norm([1.0])),
        (ValueError, lambda: clip_grad_norm([w], -1.0)),
        (ValueError, lambda: clip_grad_norm([w], float("nan"))),
        (ValueError, lambda: clip_grad_norm([w], 1.0, out=[])),
        (ValueError, lambda: clip_grad_norm([w], 1.0, out=[x])),
        (ValueError, lambda: clip_grad_norm([w], 1.0, out=[w], inplace=True)),
        (ValueError, lambda: clip_grad_norm([w.t()], 1.0, inplace=True)),
    ]
    for i, (kind, call) in enumerate(bad):
        with pytest.raises(kind):
            call()
            pytest.fail(f"call {i} was not refused")


def test_capi_rejects():
    """The C entry points report bad arguments before they touch a device."""
    from mamba2_b200 import _lib
    lib = _lib.load()
    e = _lib.EmbeddingParams(num_tokens=1, vocab=4, dim=8, weight_stride_row=8)
    assert lib.ssd_embedding(None, None) == 1 and lib.ssd_embedding(e, None) == 1      # null pointers
    e.weight_stride_row = 7
    assert lib.ssd_embedding(e, None) == 1
    e.num_tokens = 1 << 31
    assert lib.ssd_embedding(e, None) == 2
    g = _lib.EmbeddingGradParams(num_tokens=5, vocab=4, dim=8, grad_stride_row=8, out_stride_row=8, tokens=4096,
                                 grad=4096, out=4096)
    need = lib.ssd_embedding_grad_workspace_bytes(g)
    assert need > 0 and lib.ssd_embedding_grad(g, None, need, None) == 4
    assert lib.ssd_embedding_grad(g, 256, need - 1, None) == 4 and lib.ssd_embedding_grad(g, 257, need, None) == 3
    g.vocab = 0
    assert lib.ssd_embedding_grad_workspace_bytes(g) == 0 and lib.ssd_embedding_grad(g, 256, need, None) == 1
    c = _lib.LinearCeParams(tokens=2, vocab=4, dim=8, hidden_stride_row=8, weight_stride_row=8, dtype=1,
                            hidden=4096, weight=4096, targets=4096, loss=4096)
    need = lib.ssd_linear_cross_entropy_workspace_bytes(c)
    assert need > 0 and lib.ssd_linear_cross_entropy(c, None, need, None) == 4
    assert lib.ssd_linear_cross_entropy(c, 256, need - 1, None) == 4
    assert lib.ssd_linear_cross_entropy(c, 257, need, None) == 3
    for k, v, code in (("dtype", 5, 1), ("reduction", 3, 1), ("hidden_stride_row", 7, 1), ("vocab", 1 << 31, 2),
                       ("loss", None, 1), ("grad_weight_dtype", 9, 1), ("dim", 0, 1)):
        old = getattr(c, k)
        setattr(c, k, v)
        assert lib.ssd_linear_cross_entropy(c, 256, need, None) == code, k
        assert len(lib.ssd_last_error()) > 0
        setattr(c, k, old)
    t = (_lib.GradTensor * 2)()
    t[0].numel, t[0].grad, t[0].out = 10, 4096, 4096
    import ctypes
    at = ctypes.addressof(t)
    assert lib.ssd_clip_grad_norm_workspace_bytes(at, 2) == 8
    assert lib.ssd_clip_grad_norm(at, 2, 1.0, 0.0, 1, None, 256, 8, None) == 1
    assert lib.ssd_clip_grad_norm(at, 2, 1.0, 0.0, 1, 4096, None, 8, None) == 4
    assert lib.ssd_clip_grad_norm(at, 2, -1.0, 0.0, 1, 4096, 256, 8, None) == 1
    assert lib.ssd_clip_grad_norm(at, -1, 1.0, 0.0, 1, 4096, 256, 8, None) == 1
    t[0].out_dtype = 1
    assert lib.ssd_clip_grad_norm(at, 2, 1.0, 0.0, 1, 4096, 256, 8, None) == 1     # in place, two dtypes
    t[0].out = None
    assert lib.ssd_clip_grad_norm(at, 2, 1.0, 0.0, 1, 4096, 256, 8, None) == 1
