"""Numerics of the language-model operators where they can lose digits: rows, words and tokens of very
different size, confident and hopeless targets, long sums; each against float64, relative to itself.

Inputs are multiples of a power of two and few enough bits long that every logit is exact in float32 (sums
of integers below 2^24), so that what remains are the errors behind the logits.  u = 2^-24.

Gradients, per element, against the sum A of the magnitudes of its terms (|dl| |W|, or |dl|^T |X|):
- dl: exp2 (2 ulp: 2^-22), its argument (rounded: u |z|, and log2(e) as a float: u |z| / 2), the row's factor
  (4 u);
- two f16 terms per value: at most 2^-22 of it for each operand, and lo * lo: 3 * 2^-22 in all;
- adds on the tensor cores: 24 in a segment of two K blocks, each cut by up to 2 u of the sum so far; one
  rounded add per segment of 128 terms;
- what a value more than 2^16 below the largest of its row or column lacks: 2^-39 of the largest, per term.
"""
import math

import pytest
import torch

from mamba2_b200 import clip_grad_norm, embedding_grad, linear_cross_entropy, linear_cross_entropy_grad

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
DT = {"f32": torch.float32, "bf16": torch.bfloat16}


@pytest.fixture(autouse=True)
def _need_gpu():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")


def ints(shape, bits, seed, shift):
    """Integers of `bits` bits (sign included) times 2^-shift, as float64."""
    g = torch.Generator().manual_seed(seed)
    return torch.randint(-2 ** (bits - 1), 2 ** (bits - 1), shape, generator=g).double() * 2.0 ** -shift


def reference(x, w, y, coef):
    """float64: losses, lse, dl (times coef per token)."""
    s = x @ w.t()
    lse = torch.logsumexp(s, 1)
    rows = torch.arange(len(y))
    dl = torch.exp(s - lse[:, None])
    # p - 1 of the target from the others' sum, which keeps its digits where p is near 1
    others = torch.where(torch.nn.functional.one_hot(y, w.shape[0]).bool(), torch.zeros_like(dl), dl).sum(1)
    dl[rows, y] = -others
    t = s[rows, y]
    rest = s.clone()
    rest[rows, y] = -math.inf
    loss = torch.log1p(torch.exp(torch.logsumexp(rest, 1) - t))
    return loss, lse, dl * coef[:, None], s


def grad_constant(k, s):
    """c of |error| <= c A for a sum of k terms of dl; s are the logits."""
    z = float((s - s.max(1, keepdim=True).values).abs().max()) * 1.4427
    return 2.0 ** -22 + 1.5 * U * z + 4 * U + 3 * 2.0 ** -22 + 24 * 2 * U + (k / 128 + 1) * U + 4 * U


def check_grad(got, dl, m, s):
    """got against dl @ m, element by element."""
    k = dl.shape[1]
    term = dl.abs().max(1, keepdim=True).values * m.abs().max()
    bound = grad_constant(k, s) * (dl.abs() @ m.abs()) + k * 2.0 ** -38 * term
    err = (got.double().cpu() - dl @ m).abs()
    assert (err <= bound).all(), float((err / bound).max())


def grads(x, w, y, weights):
    return linear_cross_entropy_grad(x.float().cuda(), w.float().cuda(), y.cuda(), reduction="none",
                                     grad_loss=weights.float().cuda(), check_status=True)


# ---- nothing but the target, and targets without mass -------------------------------------------
@pytest.mark.parametrize("t", [1, 3, 40, 200])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("logit", [-1024.0, -3.0, 0.0, 512.0])
def test_a_vocabulary_of_one_word(t, dtype, logit):
    x, w = torch.full((t, 64), 4.0, dtype=DT[dtype]).cuda(), torch.full((1, 64), logit / 256, dtype=DT[dtype]).cuda()
    y = torch.zeros(t, dtype=torch.int64).cuda()
    loss, lse = linear_cross_entropy(x, w, y, reduction="none", return_lse=True)
    assert (loss == 0).all() and (lse == logit).all()
    loss, dx, dw = linear_cross_entropy_grad(x, w, y, reduction="sum")
    assert float(loss) == 0 and (dx == 0).all() and (dw == 0).all()


@pytest.mark.parametrize("t,dtype", [(1, "f32"), (5, "f32"), (1, "bf16"), (4, "bf16"), (40, "bf16"), (200, "bf16")])
def test_target_logit_minus_infinity(t, dtype):
    """The target has no mass: its loss is infinite, the log of the sum is that of the others."""
    x, w = ints((t, 64), 8, 0, 7), ints((30, 64), 8, 1, 7)
    x[:, 0] = 1.0
    w[3] = 0.0
    w[3, 0] = -math.inf
    y = torch.full((t,), 3)
    loss, lse = linear_cross_entropy(x.to(DT[dtype]).cuda(), w.to(DT[dtype]).cuda(), y.cuda(), reduction="none",
                                     return_lse=True)
    want = torch.logsumexp((x @ w.t())[:, [i for i in range(30) if i != 3]], 1)
    assert (loss == math.inf).all()
    assert ((lse.double().cpu() - want).abs() <= 2.0 ** -21 + 8 * U * (1 + want.abs())).all()


# ---- one large row or word beside the others ----------------------------------------------------
@pytest.mark.parametrize("t", [20, 40, 200])
@pytest.mark.parametrize("large", [2.0 ** 20, 2.0 ** 40, 2.0 ** 90])
def test_a_large_row_of_hidden_changes_no_other_loss(t, large):
    x, w = ints((t, 64), 17, 0, 14).float(), ints((300, 64), 17, 1, 18).float()
    y = torch.randint(0, 300, (t,), generator=torch.Generator().manual_seed(2))
    want = linear_cross_entropy(x.cuda(), w.cuda(), y.cuda(), reduction="none")
    x[0] *= large
    got = linear_cross_entropy(x.cuda(), w.cuda(), y.cuda(), reduction="none")
    assert torch.equal(got[1:], want[1:])


@pytest.mark.parametrize("t", [20, 40, 200])
@pytest.mark.parametrize("large", [2.0 ** 20, 2.0 ** 40, 2.0 ** 90])
def test_a_large_word_without_mass_changes_no_loss(t, large):
    x, w = ints((t, 64), 17, 0, 14).float(), ints((300, 64), 17, 1, 18).float()
    x[:, 0] = 1.0
    y = torch.randint(6, 300, (t,), generator=torch.Generator().manual_seed(2))
    w[5] = 0.0
    w[5, 0] = -1024.0
    want = linear_cross_entropy_grad(x.cuda(), w.cuda(), y.cuda(), reduction="none")
    w[5, 0] = -1024.0 * large
    got = linear_cross_entropy_grad(x.cuda(), w.cuda(), y.cuda(), reduction="none")
    assert torch.equal(got[0], want[0])
    assert all(float((a - b).norm()) <= 1e-5 * float(b.norm()) for a, b in zip(got[1:], want[1:]))


@pytest.mark.parametrize("t", [40, 200])
def test_gradients_beside_a_large_row(t):
    """hidden's rows over sixty powers of two: every row of grad_hidden relative to itself."""
    x, w = ints((t, 64), 8, 0, 7), ints((300, 64), 8, 1, 7)
    x = x * 2.0 ** -torch.arange(t).remainder(60).double()[:, None]
    y = torch.randint(0, 300, (t,), generator=torch.Generator().manual_seed(2))
    one = torch.ones(t, dtype=torch.float64)
    _, dx, dw = grads(x, w, y, one)
    _, _, dl, s = reference(x, w, y, one)
    check_grad(dx, dl, w, s)
    assert float((dw.double().cpu() - dl.t() @ x).norm()) <= 1e-5 * float((dl.t() @ x).norm())


# ---- gradients of the logits over many powers of ten --------------------------------------------
@pytest.mark.parametrize("t", [7, 40, 200, 700])
@pytest.mark.parametrize("decades", [12, 25])
def test_token_weights_over_decades(t, decades):
    x, w = ints((t, 64), 8, 0, 7), ints((513, 64), 8, 1, 7)
    g = torch.Generator().manual_seed(2)
    y = torch.randint(0, 513, (t,), generator=g)
    weights = (10.0 ** (-decades * torch.rand(t, generator=g).double())).float().double()
    weights[0] = 1.0
    _, dx, dw = grads(x, w, y, weights)
    _, _, dl, s = reference(x, w, y, weights)
    check_grad(dx, dl, w, s)
    check_grad(dw, dl.t(), x, s)


@pytest.mark.parametrize("t", [8, 40, 200])
def test_confident_rows_keep_their_gradient(t):
    """1 - p of the target from 0.9 down to 1e-12."""
    w = ints((300, 64), 8, 1, 8)
    y = torch.randint(0, 300, (t,), generator=torch.Generator().manual_seed(2))
    x = w[y] * (1 + torch.arange(t).remainder(8)).double()[:, None]
    one = torch.ones(t, dtype=torch.float64)
    loss, dx, _ = grads(x, w, y, one)
    ref, lse, dl, s = reference(x, w, y, one)
    assert float(dl.abs().sum(1).min()) < 1e-11
    check_grad(dx, dl, w, s)
    e = 2.0 ** -22 + 1.5 * U * float(s.max() - s.min()) * 1.4427 + 8 * U
    assert ((loss.double().cpu() - ref).abs() <= e * ref).all()


@pytest.mark.parametrize("t", [8, 40, 200, 700])
def test_improbable_words_keep_their_gradient(t):
    """Words with a probability below 1e-12 for every token: their rows of grad_weight, relative to themselves."""
    x, w = ints((t, 64), 8, 0, 7), ints((300, 64), 8, 1, 7)
    x[:, :32] = 127.0 / 128
    w[:40, :32] = -127.0 / 128
    y = torch.randint(40, 300, (t,), generator=torch.Generator().manual_seed(2))
    one = torch.ones(t, dtype=torch.float64)
    _, dx, dw = grads(x, w, y, one)
    _, _, dl, s = reference(x, w, y, one)
    assert float(dl[:, :40].max()) < 1e-12
    check_grad(dx, dl, w, s)
    check_grad(dw, dl.t(), x, s)


# ---- both low terms take part -------------------------------------------------------------------
@pytest.mark.parametrize("t", [40, 200])
@pytest.mark.parametrize("long", ["hidden", "weight"])
def test_f32_values_of_17_bits(t, long):
    x, w = ints((t, 64), 17, 0, 15), ints((300, 64), 2, 1, 1)
    if long == "weight":
        x, w = ints((t, 64), 2, 0, 1), ints((300, 64), 17, 1, 15)
    y = torch.randint(0, 300, (t,), generator=torch.Generator().manual_seed(2))
    one = torch.ones(t, dtype=torch.float64)
    loss, dx, dw = grads(x, w, y, one)
    ref, lse, dl, s = reference(x, w, y, one)
    got = linear_cross_entropy(x.float().cuda(), w.float().cuda(), y.cuda(), reduction="none", return_lse=True)
    bound = 2.0 ** -21 + 2 * U * s.abs().max() + 4 * U * (1 + ref.abs() + lse.abs())
    assert ((got[0].double().cpu() - ref).abs() <= bound).all() and ((got[1].double().cpu() - lse).abs() <= bound).all()
    assert ((loss.double().cpu() - ref).abs() <= bound).all()
    check_grad(dx, dl, w, s)
    check_grad(dw, dl.t(), x, s)


# ---- long sums ----------------------------------------------------------------------------------
def test_bf16_grad_hidden_has_no_bias_over_a_large_vocabulary():
    """sum_v p_v w_v over 131072 words, all terms positive: adds that cut lose the more the longer they run.
    Columns and tokens of many sizes, so that the part of the gradient along the float64 one averages the
    roundings of dl and of the result (163840 values: 2^-9 / sqrt(3) / 405 = 2.8e-6; five times that).  A
    segment of 32 K blocks has 128 adds, each cut by up to 2^-23, and 64 rounded ones join the segments."""
    t, v, d, some = 4096, 131072, 1280, 128
    g = torch.Generator(device="cuda").manual_seed(0)
    c = torch.exp2(torch.rand(d, generator=g, device="cuda"))
    w = ((torch.randn((v, d), generator=g, device="cuda") * 0.05 + 0.25) * c).bfloat16()
    w[0] = 0.0
    x = (torch.randn((t, d), generator=g, device="cuda") * 0.4 / c).bfloat16()
    weight = torch.exp2(torch.rand(t, generator=g, device="cuda"))
    y = torch.zeros(t, dtype=torch.int64, device="cuda")
    _, dx, _ = linear_cross_entropy_grad(x, w, y, reduction="none", grad_loss=weight, need_weight_grad=False,
                                         check_status=True)
    p = torch.softmax(x[:some].double() @ w.double().t(), 1) * weight[:some, None].double()
    ref = p @ w.double()
    bias = float((dx[:some].double() * ref).sum() / (ref * ref).sum()) - 1.0
    assert abs(bias) <= 128 * 2.0 ** -23 + 64 * U + 5 * 2.8e-6


# ---- ignored rows -------------------------------------------------------------------------------
@pytest.mark.parametrize("t", [2, 3, 8, 40])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("bad", [math.inf, math.nan])
def test_ignored_rows_have_no_gradient_whatever_the_weight_holds(t, dtype, bad):
    x, w = ints((t, 64), 8, 0, 7).to(DT[dtype]).cuda(), ints((30, 64), 8, 1, 7).to(DT[dtype]).cuda()
    w[7, 5] = bad
    y = torch.arange(t).cuda()
    y[0] = -100
    _, dx, _ = linear_cross_entropy_grad(x, w, y)
    assert (dx[0] == 0).all()


# ---- clipping -----------------------------------------------------------------------------------
def test_clip_refuses_out_of_another_shape():
    g = [torch.ones(6, 4).cuda(), torch.ones(5).cuda()]
    for bad in (torch.empty(4, 6), torch.empty(2, 12), torch.empty(6, 4, 1)):
        with pytest.raises(ValueError):
            clip_grad_norm(g, 1.0, out=[bad.cuda(), torch.empty(5).cuda()])
    # a piece of a flat buffer holds the values in the same order
    flat = torch.empty(29).cuda()
    got, _ = clip_grad_norm(g, 1e9, out=[flat[:24], flat[24:]])
    assert (flat == 1).all() and got[0].shape == (24,)


# ---- the paths around the scaled planes ---------------------------------------------------------
def test_f32_token_chunks():
    """More tokens than one chunk of logits holds: every chunk has powers of its own, grad_weight is summed."""
    t, v, d = 4500, 131072, 64
    g = torch.Generator(device="cuda").manual_seed(0)
    w = torch.randn(v, d, generator=g, device="cuda") / 8
    y = torch.randint(0, v, (t,), generator=g, device="cuda")
    x = torch.randn(t, d, generator=g, device="cuda") + 4 * w[y]
    weight = 10.0 ** (-6 * torch.rand(t, generator=g, device="cuda"))
    weight[t // 2:] *= 1e-6
    _, dx, dw = linear_cross_entropy_grad(x, w, y, reduction="none", grad_loss=weight, check_status=True)
    xs, ws = x.double(), w.double()
    dws, worst = torch.zeros_like(ws), 0.0
    for lo in range(0, t, 500):
        p = torch.softmax(xs[lo:lo + 500] @ ws.t(), 1)
        p[torch.arange(len(p)), y[lo:lo + 500]] -= 1
        p *= weight[lo:lo + 500, None].double()
        ref = p @ ws
        worst = max(worst, float(((dx[lo:lo + 500].double() - ref).norm(dim=1) / ref.norm(dim=1)).max()))
        dws += p.t() @ xs[lo:lo + 500]
    # a logit: 6 * 2^-22 |x| |w| / 4 of independent roundings, 24 adds cut by 2^-23 of sums up to 12; twice that
    # in a row of dl, and the product's own 1e-5
    tol = 2 * (6 * 2.0 ** -22 * 3 + 24 * 2.0 ** -23 * 12) + 1e-5
    assert worst <= tol and float((dw.double() - dws).norm() / dws.norm()) <= tol


@pytest.mark.parametrize("t", [40, 200])
def test_f32_rows_without_a_valid_target_or_weight(t):
    """An invalid target makes its own row of grad_hidden NaN (and grad_weight), and no other row; a token of
    weight zero has no gradient."""
    x, w = ints((t, 64), 8, 0, 7), ints((300, 64), 8, 1, 7)
    y = torch.randint(0, 300, (t,), generator=torch.Generator().manual_seed(2))
    one = torch.ones(t, dtype=torch.float64)
    _, _, dl, s = reference(x, w, y, one)
    bad = y.clone()
    bad[5], bad[-1] = 300, -1
    loss, dx, dw = grads(x, w, bad, one)
    keep = torch.ones(t, dtype=torch.bool)
    keep[5] = keep[-1] = False
    assert torch.isnan(loss[~keep]).all() and torch.isnan(dx[~keep]).all() and torch.isnan(dw).all()
    check_grad(dx[keep], dl[keep], w, s[keep])
    weight = one.clone()
    weight[::3] = 0.0
    _, dx, dw = grads(x, w, y, weight)
    assert (dx[::3] == 0).all()
    dl = dl * weight[:, None]
    check_grad(dx, dl, w, s)
    check_grad(dw, dl.t(), x, s)
    _, dx, dw = grads(x, w, y, 0 * one)
    assert (dx == 0).all() and (dw == 0).all()
