"""The gated linear recurrence, its gradient and its single-token step: the CUDA kernels against a plain
float64 loop over the tokens, and their refusals.

Tolerances.  u = 2^-24 and v = 2^-8 (half of torch.finfo.eps: 8 significant bits) are the largest relative errors of a rounding to float32 and bfloat16.
- The gates, in float32: sigmoid and expm1 by a few operations and approximate instructions of 2 units
  each: 16 u relative (a gate argument of magnitude 8 times log2 e is rounded by 8 u of itself, an absolute error
  of 8 * 8 u in the exponent at worst: inputs here are below 6, so 48 u); log a carries that error relatively, and so does
  b = sqrt(1 - a^2), at most half of it.  E = 64 u is taken for a and b's relative errors of log a and b.
- A state is a sum of terms a...a b w; its exponent, a sum of log a, is E of itself off.  Terms that matter have
  |sum of log a| below 20, so each is (20 + 2) E off relative to its magnitude, and each step adds a rounding u of the
  state.  So |error| <= (22 E + n u) M (a is rounded once a step as well: E holds 32 u of room for 20 of them, n u the rest) with M the same recurrence of the magnitudes |b w|, and n the steps that a
  state lives through: bounded by 64 + the 1 / (1 - a) at the slowest decay.  Plus v |y| where y is bfloat16.
- The gradients' recurrence is the same in reverse; each gradient is a product of at most 6 such factors with one
  difference: the bound is 8 times that on the product of the magnitudes.
These bounds are worst cases.  Beside them, relative 2-norms: 2e-6 in float32 (errors of different tokens do not
add up: sqrt of what is above), v in bfloat16.
"""
import math

import pytest
import torch

from mamba2_b200 import gated_recurrence, gated_recurrence_grad, gated_recurrence_update

gpu = pytest.mark.gpu
U, V = 2.0 ** -24, 2.0 ** -8
E = 64 * U
DT = {"f32": torch.float32, "bf16": torch.bfloat16}


@pytest.fixture(autouse=True)
def _need_gpu(request):
    if request.node.get_closest_marker("gpu") and not torch.cuda.is_available():
        pytest.skip("no CUDA device")


def inputs(b, L, d, dtype="f32", seed=0, keep=(0.9, 0.999)):
    g = torch.Generator().manual_seed(seed)
    x, r, i, dy = (torch.randn((b, L, d), generator=g).clamp(-6, 6).to(DT[dtype]) for _ in range(4))
    k = keep[0] + (keep[1] - keep[0]) * torch.rand(d, generator=g)
    lam = torch.log(torch.expm1(-torch.log(k) / 8.0))
    return x, r, i, lam, torch.randn((b, d), generator=g), dy, torch.randn((b, d), generator=g)


def softplus64(v):
    return torch.clamp(v, min=0) + torch.log1p(torch.exp(-v.abs()))


def loop(x, r, i, lam, h0, seq=None, scale=8.0):
    """(h, before, log a, a, b, w, starts) in float64, token by token."""
    x, r, i, lam = (t.double() for t in (x, r, i, lam))
    n, L, d = x.shape
    la = -scale * softplus64(lam) * torch.sigmoid(r)
    a = torch.exp(la)
    b, w = torch.sqrt(-torch.expm1(2 * la)), torch.sigmoid(i) * x
    starts = torch.zeros((n, L), dtype=torch.bool)
    if seq is not None and L > 1:
        starts[:, 1:] = seq[:, 1:] != seq[:, :-1]
    h = torch.zeros((n, d), dtype=torch.float64) if h0 is None else h0.double().clone()
    before, out = [], []
    for t in range(L):
        h = torch.where(starts[:, t, None], torch.zeros_like(h), h)
        before.append(h)
        h = a[:, t] * h + b[:, t] * w[:, t]
        out.append(h)
    return torch.stack(out, 1), torch.stack(before, 1), la, a, b, w, starts


def loop_grad(x, r, i, lam, h0, dy, df=None, seq=None, scale=8.0):
    """The gradients in float64, and the product of magnitudes that each is made of."""
    h, before, la, a, b, w, starts = loop(x, r, i, lam, h0, seq, scale)
    x, r, i, lam = (t.double() for t in (x, r, i, lam))
    si, sr = torch.sigmoid(i), torch.sigmoid(r)
    n, L, d = x.shape
    c = torch.zeros((n, d), dtype=torch.float64) if df is None else df.double().clone()
    cm = c.abs()
    delta, size = torch.empty_like(h), torch.empty_like(h)
    for t in range(L - 1, -1, -1):
        delta[:, t], size[:, t] = dy[:, t].double() + c, dy[:, t].double().abs() + cm
        keep = a[:, t] * (~starts[:, t, None])
        c, cm = keep * delta[:, t], keep * size[:, t]
    M, Mb = magnitude(x, r, i, lam, h0, seq, scale)
    q = torch.where(b > 0, la / torch.where(b > 0, b, torch.ones_like(b)), torch.zeros_like(b))
    m, mm = a * la * before - a * a * q * w, a * la.abs() * Mb + a * a * q.abs() * w.abs()
    rho = torch.sigmoid(lam) / softplus64(lam)
    grads = (delta * b * si, delta * m * (1 - sr), delta * b * w * (1 - si), rho * (delta * m).sum((0, 1)), c)
    sizes = (size * b * si, size * mm, size * b * w.abs(), rho * (size * mm).sum((0, 1)), cm)
    return grads, sizes


def magnitude(x, r, i, lam, h0, seq, scale):
    x, r, i, lam = (t.double() for t in (x, r, i, lam))
    h, before, *_ = loop(x.abs(), r, i, lam, None if h0 is None else h0.abs(), seq, scale)
    return h, before


def lives(lam, scale=8.0):
    """Steps that a state lives through at the slowest decay of gates around 0 (a quarter open)."""
    return 64 + 1.0 / max(1e-4, float(1 - torch.exp(-scale * softplus64(lam.double()) * 0.25).max()))


def cuda(*ts):
    return [None if t is None else t.cuda() for t in ts]


def close(got, ref, bound, dtype, norm=True):
    got = got.double().cpu()
    assert torch.isfinite(got).all()
    if dtype == "bf16":
        bound = bound + V * ref.abs() * (1 + 1e-3) + 1e-38
    worst = float(((got - ref).abs() - bound).max()) if got.numel() else 0.0
    assert worst <= 0, worst
    if norm and got.numel() and float(ref.norm()) > 0:
        rel = float((got - ref).norm() / ref.norm())
        assert rel <= (V if dtype == "bf16" else 2e-6), rel


SHAPES = [(1, 1, 1), (1, 2, 64), (2, 7, 31), (1, 8, 32), (3, 63, 65), (1, 64, 128), (2, 65, 66), (1, 129, 8),
          (1, 513, 72), (5, 200, 40), (1, 1100, 33), (2, 2049, 64)]


@gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("b,L,d", SHAPES)
def test_forward(b, L, d, dtype):
    x, r, i, lam, h0, _, _ = inputs(b, L, d, dtype, seed=L + d)
    for start in (None, h0):
        ref = loop(x, r, i, lam, start)[0]
        bound = (22 * E + lives(lam) * U) * magnitude(x, r, i, lam, start, None, 8.0)[0]
        y, final = gated_recurrence(*cuda(x, r, i, lam), initial_state=None if start is None else start.cuda(),
                                    return_final_state=True)
        assert y.dtype == DT[dtype] and final.dtype == torch.float32
        close(y, ref, bound, dtype)
        close(final, ref[:, -1], bound[:, -1], "f32")


@gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("b,L,d", SHAPES)
def test_gradients(b, L, d, dtype):
    x, r, i, lam, h0, dy, df = inputs(b, L, d, dtype, seed=L + 3 * d)
    for start, last in ((None, None), (h0, df)):
        refs, sizes = loop_grad(x, r, i, lam, start, dy, last)
        args = cuda(x, r, i, lam, dy)
        kw = dict(initial_state=None if start is None else start.cuda(), grad_final_state=None if last is None else last.cuda())
        got = gated_recurrence_grad(*args, **kw)
        *_, points = gated_recurrence(*args[:4], initial_state=kw["initial_state"], return_checkpoints=True)
        again = gated_recurrence_grad(*args, **kw, checkpoints=points)
        assert (got[4] is None) == (start is None)
        c = 8 * (22 * E + lives(lam) * U)
        for k in range(5):
            if got[k] is None:
                continue
            assert torch.equal(got[k], again[k])
            close(got[k], refs[k], c * sizes[k], dtype if k < 3 else "f32", norm=k < 3)


@gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("ends", [(1,), (8,), (7, 9), (64,), (63, 64, 65), (1, 2, 3, 4), (100, 164, 228, 500), (510, 511)])
def test_packed_sequences(ends, dtype):
    """Every start position of a tile, a warp and a cluster; each sequence alone gives the same values."""
    b, L, d = 2, 512, 40
    x, r, i, lam, h0, dy, df = inputs(b, L, d, dtype, seed=sum(ends))
    seq = torch.zeros((b, L), dtype=torch.int32)
    for e in ends:
        seq[0, e:] += 1
    seq[1] = 7          # the other row is one sequence
    ref = loop(x, r, i, lam, h0, seq)[0]
    bound = (22 * E + lives(lam) * U) * magnitude(x, r, i, lam, h0, seq, 8.0)[0]
    args = cuda(x, r, i, lam)
    y, final = gated_recurrence(*args, initial_state=h0.cuda(), seq_idx=seq.cuda(), return_final_state=True)
    close(y, ref, bound, dtype)
    close(final, ref[:, -1], bound[:, -1], "f32")
    refs, sizes = loop_grad(x, r, i, lam, h0, dy, df, seq)
    got = gated_recurrence_grad(*args, dy.cuda(), initial_state=h0.cuda(), seq_idx=seq.cuda(), grad_final_state=df.cuda())
    for k in range(5):
        close(got[k], refs[k], 8 * (22 * E + lives(lam) * U) * sizes[k], dtype if k < 3 else "f32", norm=k < 3)


@gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("near", [True, False])
@pytest.mark.parametrize("b,L,d", [(1, 2000, 64), (1, 4000, 64), (2, 2049, 64), (3, 1500, 256), (16, 300, 1024)])
def test_packed_sequences_of_few_channels(b, L, d, near, dtype):
    """Few rows and channels take CTAs of 8 and 16 warps in clusters of up to 16, where no pass has more than one turn or a few; sequences
    start on both sides of their tiles' ends and anywhere between.  Decays that leave a near 1, and larger ones."""
    x, r, i, lam, h0, dy, df = inputs(b, L, d, dtype, seed=L + b)
    if not near:
        lam = torch.linspace(-3.0, 1.0, d)
    g = torch.Generator().manual_seed(26)
    ends = torch.rand((b, L), generator=g) < 0.004
    ends[0, ::256], ends[-1, 127::256], ends[0, 129::512], ends[:, 0] = True, True, True, False
    seq = torch.cumsum(ends, 1).to(torch.int32)
    n = 22 * E + lives(lam) * U
    y, final = gated_recurrence(*cuda(x, r, i, lam), initial_state=h0.cuda(), seq_idx=seq.cuda(), return_final_state=True, check_status=True)
    ref, bound = loop(x, r, i, lam, h0, seq)[0], n * magnitude(x, r, i, lam, h0, seq, 8.0)[0]
    close(y, ref, bound, dtype)
    close(final, ref[:, -1], bound[:, -1], "f32")
    refs, sizes = loop_grad(x, r, i, lam, h0, dy, df, seq)
    got = gated_recurrence_grad(*cuda(x, r, i, lam, dy), initial_state=h0.cuda(), seq_idx=seq.cuda(), grad_final_state=df.cuda(), check_status=True)
    for k in range(5):
        close(got[k], refs[k], 8 * n * sizes[k], dtype if k < 3 else "f32", norm=k < 3)


@gpu
def test_every_token_its_own_sequence():
    x, r, i, lam, h0, dy, _ = inputs(1, 130, 32, seed=5)
    seq = torch.arange(130, dtype=torch.int64)[None]
    _, _, _, _, b, w, _ = loop(x, r, i, lam, None)
    y = gated_recurrence(*cuda(x, r, i, lam), seq_idx=seq.cuda())
    close(y, b * w, 4 * E * (b * w).abs(), "f32")


@gpu
def test_ids_of_64_bits():
    """Ids that differ by a multiple of 2^32, and negative ones."""
    x, r, i, lam, *_ = (t.cuda() for t in inputs(2, 90, 32, seed=4))
    ids = torch.zeros((2, 90), dtype=torch.int64, device="cuda")
    ids[0, 40:], ids[0, 70:], ids[1, 10:] = 1 << 32, -(1 << 40), -1
    small = torch.zeros((2, 90), dtype=torch.int32, device="cuda")
    small[0, 40:], small[0, 70:], small[1, 10:] = 5, -7, 3
    assert torch.equal(gated_recurrence(x, r, i, lam, seq_idx=ids), gated_recurrence(x, r, i, lam, seq_idx=small))
    one = torch.zeros((2, 1), dtype=torch.int64, device="cuda")
    assert torch.equal(gated_recurrence(x[:, :1], r[:, :1], i[:, :1], lam, seq_idx=one), gated_recurrence(x, r, i, lam)[:, :1])


@gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_values_do_not_cross_sequences(dtype):
    """NaN and infinities in one packed sequence, in the state before it and in the gradient."""
    x, r, i, lam, h0, dy, _ = inputs(1, 300, 48, dtype, seed=6)
    seq = torch.zeros((1, 300), dtype=torch.int32)
    seq[0, 100:200], seq[0, 200:] = 1, 2
    clean = cuda(x, r, i, lam, dy)
    y0 = gated_recurrence(*clean[:4], seq_idx=seq.cuda())
    g0 = gated_recurrence_grad(*clean, seq_idx=seq.cuda())
    for bad in (float("nan"), float("inf"), -float("inf")):
        for where in range(4):
            ts = [t.clone() for t in (x, r, i, dy)]
            ts[where][0, 150] = bad
            args = cuda(ts[0], ts[1], ts[2], lam)
            y = gated_recurrence(*args, seq_idx=seq.cuda())
            g = gated_recurrence_grad(*args, ts[3].cuda(), seq_idx=seq.cuda())
            for keep in (slice(0, 100), slice(200, 300)):
                assert torch.equal(y[:, keep], y0[:, keep])
                for k in range(3):
                    assert torch.equal(g[k][:, keep], g0[k][:, keep])
    h = torch.full((1, 48), float("nan"))
    y = gated_recurrence(*clean[:4], initial_state=h.cuda(), seq_idx=seq.cuda())
    assert torch.isnan(y[:, :100]).all() and torch.equal(y[:, 100:], y0[:, 100:])


@gpu
def test_saturated_gates():
    """Gates that are all but closed or open, and channels that keep everything or nothing."""
    b, L, d = 1, 200, 8
    x, r, i, lam, h0, dy, df = inputs(b, L, d, seed=7)
    r[0, 10:40], r[0, 60:90], i[0, 100:120], i[0, 130:150] = -200.0, 200.0, -200.0, 200.0
    lam = torch.tensor([-200.0, -40.0, -10.0, 0.0, 5.0, 30.0, 100.0, -120.0])
    refs, _ = loop_grad(x, r, i, lam, h0, dy, df)
    ref = loop(x, r, i, lam, h0)[0]
    y = gated_recurrence(*cuda(x, r, i, lam), initial_state=h0.cuda())
    got = gated_recurrence_grad(*cuda(x, r, i, lam, dy), initial_state=h0.cuda(), grad_final_state=df.cuda())
    assert torch.isfinite(y).all() and all(torch.isfinite(g).all() for g in got)
    assert float((y.double().cpu() - ref).norm() / ref.norm()) < 1e-5
    for k in (0, 2, 4):
        assert float((got[k].double().cpu() - refs[k]).norm() / refs[k].norm()) < 1e-5
    # the decay's gradients, channel by channel where float32 can hold the rate (k above 1e-38)
    for c in (1, 2, 3, 4, 5, 6):
        e = float((got[1][..., c].double().cpu() - refs[1][..., c]).norm())
        assert e <= 1e-5 * float(refs[1][..., c].norm()) + 1e-30, c


FAR = [-104.0, -1e3, -1.2e6, -1e7, -1e9, torch.finfo(torch.float32).min, -math.inf]


@gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_decays_that_keep_everything(dtype):
    """softplus(decay) below float32's smallest number: a is 1 and b is 0 (the formula's b is below 1e-21), whatever the gates."""
    n, b, L = len(FAR), 2, 70
    x, r, i, _, h0, dy, df = inputs(b, L, 3 * n, dtype, seed=21)
    r[0, 10:20], r[1, 30:40] = 200.0, -200.0
    lam = torch.tensor([v for f in FAR for v in (f, -5.0, f)])     # beside channels that decay, alike in both lanes of a pair
    ref = loop(x, r, i, lam, h0)[0]
    bound = (22 * E + lives(torch.tensor([-5.0])) * U) * magnitude(x, r, i, lam, h0, None, 8.0)[0]
    y, final = gated_recurrence(*cuda(x, r, i, lam), initial_state=h0.cuda(), return_final_state=True)
    close(y, ref, bound + 1e-18, dtype)
    close(final, ref[:, -1], bound[:, -1] + 1e-18, "f32")
    new, one = gated_recurrence_update(h0.cuda(), *cuda(x[:, 0], r[:, 0], i[:, 0], lam))
    close(new, ref[:, 0], 24 * E * magnitude(x, r, i, lam, h0, None, 8.0)[0][:, 0] + 1e-18, "f32")
    close(one, ref[:, 0], 24 * E * magnitude(x, r, i, lam, h0, None, 8.0)[0][:, 0] + 1e-18, dtype)
    got = gated_recurrence_grad(*cuda(x, r, i, lam, dy), initial_state=h0.cuda(), grad_final_state=df.cuda())
    keep = torch.tensor([v != -5.0 for v in lam.tolist()])
    assert torch.equal(final.cpu()[:, keep], h0[:, keep]) and torch.equal(new.cpu()[:, keep], h0[:, keep])
    for k in range(3):
        assert float(got[k][..., keep].abs().max()) <= 1e-18
    assert float(got[3][keep].abs().max()) <= 1e-18
    want = dy.double().sum(1) + df.double()
    close(got[4].cpu()[:, keep], want[:, keep], (L + 1) * U * (dy.double().abs().sum(1) + df.double().abs())[:, keep], "f32", norm=False)
    short = [g.cpu()[..., ~keep] for g in got[:3]]
    refs, sizes = loop_grad(x[..., ~keep], r[..., ~keep], i[..., ~keep], lam[~keep], h0[:, ~keep], dy[..., ~keep], df[:, ~keep])
    for k in range(3):
        # (2^-126: the closed gate's sigmoid(-200) = 1e-87 and its root 1e-44, and with them their gradients, are below float32's range)
        close(short[k], refs[k], 8 * (22 * E + lives(lam[~keep]) * U) * sizes[k] + 2.0 ** -126, dtype, norm=False)


@gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("packed", [False, True])
def test_decays_that_keep_nothing(dtype, packed):
    """scale * softplus(decay) beyond float32: a is 0 and b is 1, so that a token gives w = sigmoid(i) x, and every gradient is
    that token's own.  (70 tokens end inside a tile.)"""
    b, L = 2, 70
    most = torch.finfo(torch.float32).max
    lam = torch.tensor([most, 1e38, math.inf, 5e37] * 3 + [most])
    x, r, i, _, h0, dy, df = inputs(b, L, lam.numel(), dtype, seed=22)
    seq = torch.zeros((b, L), dtype=torch.int32)
    seq[0, 33:] = 1
    kw = dict(initial_state=h0.cuda(), seq_idx=seq.cuda() if packed else None)
    si = torch.sigmoid(i.double())
    w = si * x.double()
    y, final = gated_recurrence(*cuda(x, r, i, lam), return_final_state=True, **kw)
    close(y, w, E * w.abs(), dtype)
    close(final, w[:, -1], E * w[:, -1].abs(), "f32")
    for t in (0, L - 1):
        new, one = gated_recurrence_update(h0.cuda(), *cuda(x[:, t], r[:, t], i[:, t], lam))
        close(new, w[:, t], E * w[:, t].abs(), "f32")
        close(one, w[:, t], E * w[:, t].abs(), dtype)
    got = gated_recurrence_grad(*cuda(x, r, i, lam, dy), grad_final_state=df.cuda(), **kw)
    delta = dy.double().clone()
    delta[:, -1] += df.double()
    close(got[0], delta * si, E * (delta * si).abs() + 2 * U * delta.abs(), dtype)
    close(got[2], delta * w * (1 - si), 4 * E * (delta * w).abs(), dtype)
    for k in (1, 3, 4):
        assert float(got[k].abs().max()) == 0


@gpu
def test_decays_that_keep_nothing_behind_a_closed_gate():
    """A gate whose sigmoid is zero in float32 keeps the state, whatever the decay."""
    x, r, i, _, h0, *_ = inputs(1, 40, 4, seed=23)
    lam = torch.full((4,), torch.finfo(torch.float32).max)
    r[:, 5:] = -math.inf
    y, final = gated_recurrence(*cuda(x, r, i, lam), initial_state=h0.cuda(), return_final_state=True)
    assert torch.isfinite(y).all() and torch.equal(final, y[:, 4]) and torch.equal(y[:, 5:], y[:, 4:5].expand(1, 35, 4))
    state, _ = gated_recurrence_update(h0.cuda(), *cuda(x[:, 5], r[:, 5], i[:, 5], lam))
    assert torch.equal(state.cpu(), h0)


@gpu
def test_gradient_of_the_decay_channel_by_channel():
    """Far negative, moderate and large decays, gates that are all but closed or open: each channel on its own size."""
    b, L, d = 2, 200, 8
    x, r, i, lam, h0, dy, df = inputs(b, L, d, seed=24)
    r[0, 10:40], r[0, 60:90], i[0, 100:120], i[0, 130:150] = -200.0, 200.0, -200.0, 200.0
    lam = torch.tensor([-80.0, -40.0, -10.0, -3.0, 0.0, 5.0, 30.0, 100.0])
    refs, sizes = loop_grad(x, r, i, lam, h0, dy, df)
    got = gated_recurrence_grad(*cuda(x, r, i, lam, dy), initial_state=h0.cuda(), grad_final_state=df.cuda())[3].double().cpu()
    for c in range(d):
        # (no state lives through more than the 200 tokens)
        assert abs(float(got[c] - refs[3][c])) <= 8 * (22 * E + L * U) * float(sizes[3][c]) + 1e-30, c


@gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_gradient_of_the_decay_over_many_tokens(dtype):
    """Summands that are all alike, where every addition to a running sum rounds the same way.  Against the same summands of a short
    row, so that nothing but the sums differs.  8 summands of a turn are added up in float32 (8 u at most, in both), the turns by a compensated
    sum (2 u), and warps and CTAs join by 16 additions at most (16 u in both); a state or a gradient that another order of steps rounds
    otherwise moves a summand by 8 u: 96 u takes that in.  (One running sum of 4096 would be off by up to 2000 u.)"""
    L, d = 16384, 18944 if dtype == "f32" else 37888
    g = torch.Generator(device="cuda").manual_seed(25)

    def row(lo, hi):
        return (lo + (hi - lo) * torch.rand((1, 1, d), generator=g, device="cuda")).to(DT[dtype])

    x, r, i, dy = row(0.5, 1.5), row(-1, 1), row(-1, 1), row(0.5, 1.5)
    lam = torch.linspace(-1.5, 0.0, d, device="cuda")    # a between 0.1 and 0.6 of the state is kept

    def rows(n):
        return [t.expand(1, n, d) for t in (x, r, i)] + [lam]

    # the state, and the gradient that reaches it, where neither moves any more
    h = gated_recurrence(*rows(256), return_final_state=True)[1]
    c = gated_recurrence_grad(*rows(256), dy.expand(1, 256, d), initial_state=h)[4]
    sums = [gated_recurrence_grad(*rows(n), dy.expand(1, n, d), initial_state=h, grad_final_state=c)[3].double() / n for n in (64, L)]
    assert float(sums[0].abs().min()) > 1e-3
    assert float(((sums[1] - sums[0]) / sums[0]).abs().max()) <= 96 * U


@gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_strides_and_broadcasts(dtype):
    """Slices of one fused projection, odd starts, transposed tokens, one row for all tokens."""
    b, L, d = 2, 150, 40
    g = torch.Generator().manual_seed(8)
    fused = torch.randn((b, L, 3 * d + 5), generator=g).to(DT[dtype]).cuda()
    lam = torch.linspace(-6, -3, d).cuda()
    dy = torch.randn((b, L, d), generator=g).to(DT[dtype]).cuda()
    n = 22 * E + lives(lam.cpu()) * U
    for at in (0, 1, 2, 4, 5):      # (starts that are not on 16 bytes go another way through the kernels)
        x, r, i = (fused[..., at + k * d:at + (k + 1) * d] for k in range(3))
        cpu = [t.cpu() for t in (x, r, i, lam)]
        close(gated_recurrence(x, r, i, lam), loop(*cpu, None)[0], n * magnitude(*cpu, None, None, 8.0)[0], dtype)
        refs, sizes = loop_grad(*cpu, None, dy.cpu())
        for k, p in enumerate(gated_recurrence_grad(x, r, i, lam, dy)[:4]):
            close(p, refs[k], 8 * n * sizes[k], dtype if k < 3 else "f32", norm=k < 3)
    x, r, i = (fused[..., k * d:(k + 1) * d].contiguous() for k in range(3))
    xt = x.transpose(0, 1).contiguous().transpose(0, 1)
    assert torch.equal(gated_recurrence(xt, r, i, lam), gated_recurrence(x, r, i, lam))
    one = r[:, :1].expand(b, L, d)
    assert torch.equal(gated_recurrence(x, one, i, lam), gated_recurrence(x, one.contiguous(), i, lam))
    chan = x.transpose(1, 2).contiguous().transpose(1, 2)
    assert torch.equal(gated_recurrence(chan, r, i, lam), gated_recurrence(x, r, i, lam))
    dy = torch.ones((), dtype=DT[dtype], device="cuda").expand(b, L, d)
    for p, q in zip(gated_recurrence_grad(x, r, i, lam, dy)[:4], gated_recurrence_grad(x, r, i, lam, dy.contiguous())[:4]):
        assert torch.equal(p, q)


@gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("packed", [False, True])
def test_rows_that_start_anywhere(dtype, packed):
    """Views of buffers that hold NaN around them, every start of a row within 16 bytes, one and several groups of channels."""
    b, L = 2, 83
    for d in (1, 27, 57, 113):
        x, r, i, lam, h0, dy, df = inputs(b, L, d, seed=d)
        seq = torch.tensor([0] * 5 + [1] + [2] * 30 + [3] * 47, dtype=torch.int32).expand(b, L).contiguous() if packed else None
        data = [t.to(DT[dtype]) for t in (x, r, i, dy)]
        n = 22 * E + lives(lam) * U
        close(gated_recurrence(*cuda(*data[:3], lam), initial_state=h0.cuda(), seq_idx=cuda(seq)[0]),
              loop(*data[:3], lam, h0, seq)[0], n * magnitude(*data[:3], lam, h0, seq, 8.0)[0], dtype)
        kw = dict(initial_state=h0.cuda(), seq_idx=cuda(seq)[0])
        whole = cuda(*data)
        y, final, points = gated_recurrence(*whole[:3], lam.cuda(), return_final_state=True, return_checkpoints=True, **kw)
        grads = gated_recurrence_grad(*whole[:3], lam.cuda(), whole[3], grad_final_state=df.cuda(), checkpoints=points, **kw)
        refs, sizes = loop_grad(*data[:3], lam, h0, data[3], df, seq)
        for k, q in enumerate(grads):
            close(q, refs[k], 8 * n * sizes[k], dtype if k < 3 else "f32", norm=k < 3)
        for at in range(9):
            views = []
            for k, t in enumerate(whole):
                wide = torch.full((b, L, d + 16 + k), float("nan"), dtype=DT[dtype], device="cuda")
                view = wide[..., (at + 3 * k) % 9:][..., :d]
                view.copy_(t)
                views.append(view)
            for p, q in zip(gated_recurrence(*views[:3], lam.cuda(), return_final_state=True, return_checkpoints=True, **kw), (y, final, points)):
                assert torch.equal(p, q), (d, at)
            for p, q in zip(gated_recurrence_grad(*views[:3], lam.cuda(), views[3], grad_final_state=df.cuda(), checkpoints=points, **kw), grads):
                assert torch.equal(p, q), (d, at)


@gpu
@pytest.mark.parametrize("b,L,d", [(1, 777, 64), (64, 70, 64), (1, 4000, 2048), (7, 300, 5000)])
def test_cluster_sizes_agree_with_halves(b, L, d):
    """A sequence in two calls, the state carried between them: other clusters, other tiles."""
    x, r, i, lam, h0, dy, df = (t.cuda() for t in inputs(b, L, d, seed=9))
    y, final = gated_recurrence(x, r, i, lam, initial_state=h0, return_final_state=True)
    at = L // 3 + 1
    y1, mid = gated_recurrence(x[:, :at], r[:, :at], i[:, :at], lam, initial_state=h0, return_final_state=True)
    y2, end = gated_recurrence(x[:, at:], r[:, at:], i[:, at:], lam, initial_state=mid, return_final_state=True)
    scale = float(y.abs().max())
    assert float((torch.cat([y1, y2], 1) - y).abs().max()) <= 1e-5 * scale
    assert float((end - final).abs().max()) <= 1e-5 * scale
    whole = gated_recurrence_grad(x, r, i, lam, dy, initial_state=h0, grad_final_state=df)
    second = gated_recurrence_grad(x[:, at:], r[:, at:], i[:, at:], lam, dy[:, at:], initial_state=mid, grad_final_state=df)
    first = gated_recurrence_grad(x[:, :at], r[:, :at], i[:, :at], lam, dy[:, :at], initial_state=h0, grad_final_state=second[4])
    for k in range(3):
        joined = torch.cat([first[k], second[k]], 1)
        assert float((joined - whole[k]).norm() / whole[k].norm()) <= 4e-6
    assert float((first[3] + second[3] - whole[3]).norm() / whole[3].norm()) <= 2e-5
    assert float((first[4] - whole[4]).norm() / whole[4].norm()) <= 4e-6


@gpu
@pytest.mark.parametrize("b,L,d", [(1, 40, 6), (2, 70, 3)])
def test_gradients_against_differences(b, L, d):
    """Central differences of the float64 loop, along random directions of every input."""
    x, r, i, lam, h0, dy, df = inputs(b, L, d, seed=10)
    got = [g.double().cpu() for g in gated_recurrence_grad(*cuda(x, r, i, lam, dy), initial_state=h0.cuda(), grad_final_state=df.cuda())]

    def value(ts):
        h = loop(*ts)[0]
        return float((h * dy.double()).sum() + (h[:, -1] * df.double()).sum())

    g = torch.Generator().manual_seed(11)
    base = [t.double() for t in (x, r, i, lam, h0)]
    for k in range(5):
        v = torch.randn(base[k].shape, generator=g, dtype=torch.float64)
        eps = 1e-5
        hi, lo = list(base), list(base)
        hi[k], lo[k] = base[k] + eps * v, base[k] - eps * v
        want = (value(hi) - value(lo)) / (2 * eps)
        have = float((got[k] * v).sum())
        assert abs(have - want) <= 1e-5 * float((got[k] * v).abs().sum()) + 1e-6, k


@gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("b,d", [(1, 1), (1, 4), (3, 5), (2, 1000), (300, 64), (70000, 4)])
def test_update(b, d, dtype):
    x, r, i, lam, h0, _, _ = inputs(b, 1, d, dtype, seed=b + d)
    ref = loop(x, r, i, lam, h0)[0][:, 0]
    bound = 24 * E * magnitude(x, r, i, lam, h0, None, 8.0)[0][:, 0]
    state = h0.cuda()
    new, y = gated_recurrence_update(state, *cuda(x[:, 0], r[:, 0], i[:, 0], lam))
    assert torch.equal(state.cpu(), h0) and new.data_ptr() != state.data_ptr()
    close(y, ref, bound, dtype)
    close(new, ref, bound, "f32")
    same, y2 = gated_recurrence_update(state, *cuda(x[:, 0], r[:, 0], i[:, 0], lam), inplace=True)
    assert same is state and torch.equal(same, new) and torch.equal(y, y2)


@gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_prefill_then_steps(dtype):
    """A prefill's final state, stepped on, gives what the longer sequence gives."""
    x, r, i, lam, h0, _, _ = inputs(3, 90, 40, dtype, seed=12)
    xc, rc, ic, lc = cuda(x, r, i, lam)
    y, final = gated_recurrence(xc, rc, ic, lc, initial_state=h0.cuda(), return_final_state=True)
    got, state = gated_recurrence(xc[:, :70], rc[:, :70], ic[:, :70], lc, initial_state=h0.cuda(), return_final_state=True)
    steps = [got]
    for t in range(70, 90):
        state, h = gated_recurrence_update(state, xc[:, t], rc[:, t], ic[:, t], lc, inplace=True)
        steps.append(h[:, None])
    M = magnitude(x, r, i, lam, h0, None, 8.0)[0]
    bound = 2 * (22 * E + lives(lam) * U) * M + (0 if dtype == "f32" else 2 * V) * M
    assert float(((torch.cat(steps, 1).double() - y.double()).cpu().abs() - bound).max()) <= 0
    assert float(((state.double() - final.double()).cpu().abs() - 2 * (22 * E + lives(lam) * U) * M[:, -1]).max()) <= 0


@gpu
def test_scale_zero_keeps_the_state():
    x, r, i, lam, h0, dy, _ = inputs(2, 70, 8, seed=13)
    y = gated_recurrence(*cuda(x, r, i, lam), scale=0.0, initial_state=h0.cuda())
    assert torch.equal(y.cpu(), h0[:, None].expand(2, 70, 8))
    g = gated_recurrence_grad(*cuda(x, r, i, lam, dy), scale=0.0, initial_state=h0.cuda())
    assert all(float(t.abs().max()) == 0 for t in g[:4])
    assert torch.allclose(g[4].cpu(), dy.sum(1), rtol=1e-5, atol=1e-5)


@gpu
def test_empty():
    for b, L in ((0, 5), (2, 0)):
        x, r, i, dy = (torch.zeros((b, L, 8), device="cuda") for _ in range(4))
        lam, h0 = torch.zeros(8, device="cuda"), torch.ones((b, 8), device="cuda")
        y, final, points = gated_recurrence(x, r, i, lam, initial_state=h0, return_final_state=True, return_checkpoints=True)
        assert y.shape == (b, L, 8) and torch.equal(final, h0) and points.numel() == 0
        g = gated_recurrence_grad(x, r, i, lam, dy, initial_state=h0, grad_final_state=2 * h0)
        assert float(g[3].abs().max()) == 0 and torch.equal(g[4], 2 * h0)
    assert float(gated_recurrence(torch.zeros((2, 0, 8), device="cuda"), torch.zeros((2, 0, 8), device="cuda"),
                                  torch.zeros((2, 0, 8), device="cuda"), torch.zeros(8, device="cuda"),
                                  return_final_state=True)[1].abs().max()) == 0
    z = torch.zeros((0, 8), device="cuda")
    assert gated_recurrence_update(z, z, z, z, torch.zeros(8, device="cuda"))[1].shape == (0, 8)


@gpu
def test_equal_calls_give_equal_bits_and_graphs_replay():
    x, r, i, lam, h0, dy, df = (t.cuda() for t in inputs(2, 3000, 192, "bf16", seed=14))

    def step():
        y, final, points = gated_recurrence(x, r, i, lam, initial_state=h0, return_final_state=True, return_checkpoints=True)
        return (y, final) + gated_recurrence_grad(x, r, i, lam, dy, initial_state=h0, checkpoints=points) + \
            gated_recurrence_grad(x, r, i, lam, dy, initial_state=h0, grad_final_state=df)

    want = step()
    assert all(torch.equal(p, q) for p, q in zip(step(), want))
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    torch.cuda.current_stream().wait_stream(s)
    graphs = []
    for _ in range(2):     # two graphs, replayed in turn
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = step()
        graphs.append((graph, got))
    for _ in range(2):
        for graph, got in graphs:
            for t in got:
                t.fill_(float("nan"))
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(p, q) for p, q in zip(got, want))
    x.copy_(torch.randn_like(x, dtype=torch.float32))
    graphs[0][0].replay()
    fresh = step()
    torch.cuda.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(graphs[0][1], fresh))


@gpu
def test_two_streams_at_once():
    sets = [tuple(t.cuda() for t in inputs(1, 5000, 256, "bf16", seed=s)) for s in (15, 16)]
    want = [gated_recurrence_grad(*t[:4], t[5], initial_state=t[4]) for t in sets]
    streams = [torch.cuda.Stream() for _ in sets]
    torch.cuda.synchronize()
    got = [None, None]
    for _ in range(3):
        for k, (s, t) in enumerate(zip(streams, sets)):
            with torch.cuda.stream(s):
                got[k] = gated_recurrence_grad(*t[:4], t[5], initial_state=t[4])
    torch.cuda.synchronize()
    for p, q in zip(got, want):
        assert all(torch.equal(a, b) for a, b in zip(p, q))


@gpu
@pytest.mark.slow
def test_past_32_bit_offsets():
    """More than 2^31 values: the last rows equal those of a short call."""
    b, L, d = 1, 2_200_000, 1024
    lam = torch.full((d,), -4.0, device="cuda")
    x = torch.empty((b, L, d), dtype=torch.bfloat16, device="cuda")
    for lo in range(0, L, 100_000):
        x[:, lo:lo + 100_000].normal_()
    seq = torch.zeros((b, L), dtype=torch.int32, device="cuda")
    seq[:, L - 300:] = 1
    y, final = gated_recurrence(x, x, x, lam, seq_idx=seq, return_final_state=True)
    tail = x[:, L - 300:]
    want, end = gated_recurrence(tail, tail, tail, lam, return_final_state=True)
    assert float((y[:, L - 300:].float() - want.float()).norm() / want.float().norm()) <= V
    assert float((final - end).norm() / end.norm()) <= 2e-6
    del y
    g = gated_recurrence_grad(x, x, x, lam, x, seq_idx=seq)
    short = gated_recurrence_grad(tail, tail, tail, lam, tail)
    for k in range(3):
        assert float((g[k][:, L - 300:].float() - short[k].float()).norm() / short[k].float().norm()) <= 2 * V


def test_refusals_need_no_gpu():
    x, lam = torch.zeros((1, 4, 8)), torch.zeros(8)
    with pytest.raises(ValueError, match="CUDA"):
        gated_recurrence(x, x, x, lam)
    with pytest.raises(ValueError, match="CUDA"):
        gated_recurrence_grad(x, x, x, lam, x)
    with pytest.raises(TypeError, match="torch.Tensor"):
        gated_recurrence(x.numpy(), x, x, lam)
    with pytest.raises(TypeError, match="float32"):
        gated_recurrence_update(torch.zeros((1, 8), dtype=torch.float64), x[:, 0], x[:, 0], x[:, 0], lam)
    with pytest.raises(ValueError, match="CUDA"):
        gated_recurrence_update(torch.zeros((1, 8)), x[:, 0], x[:, 0], x[:, 0], lam)


@gpu
def test_refusals():
    x, lam, h = torch.zeros((2, 70, 8), device="cuda"), torch.zeros(8, device="cuda"), torch.zeros((2, 8), device="cuda")
    cases = [
        (ValueError, lambda: gated_recurrence(x[0], x, x, lam)),
        (ValueError, lambda: gated_recurrence(x, x[:, :5], x, lam)),
        (ValueError, lambda: gated_recurrence(x, x, x[..., :4], lam)),
        (ValueError, lambda: gated_recurrence(x, x, x, lam[:4])),
        (ValueError, lambda: gated_recurrence(x, x, x, lam.cpu())),
        (TypeError, lambda: gated_recurrence(x, x.bfloat16(), x, lam)),
        (TypeError, lambda: gated_recurrence(x.half(), x.half(), x.half(), lam)),
        (ValueError, lambda: gated_recurrence(x, x, x, lam, scale=-1.0)),
        (ValueError, lambda: gated_recurrence(x, x, x, lam, scale=float("nan"))),
        (ValueError, lambda: gated_recurrence(x, x, x, lam, scale=float("inf"))),
        (ValueError, lambda: gated_recurrence(x, x, x, lam, initial_state=h[:1])),
        (ValueError, lambda: gated_recurrence(x, x, x, lam, initial_state=h.cpu())),
        (ValueError, lambda: gated_recurrence(x, x, x, lam, seq_idx=torch.zeros((2, 69), dtype=torch.int32, device="cuda"))),
        (TypeError, lambda: gated_recurrence(x, x, x, lam, seq_idx=torch.zeros((2, 70), device="cuda"))),
        (ValueError, lambda: gated_recurrence(x[..., :0], x[..., :0], x[..., :0], lam[:0])),
        (ValueError, lambda: gated_recurrence_grad(x, x, x, lam, x[:1])),
        (TypeError, lambda: gated_recurrence_grad(x, x, x, lam, x.bfloat16())),
        (ValueError, lambda: gated_recurrence_grad(x, x, x, lam, x, checkpoints=torch.zeros((2, 1, 8), device="cuda"))),
        (ValueError, lambda: gated_recurrence_grad(x, x, x, lam, x, checkpoints=torch.zeros((2, 3, 8), device="cuda").bfloat16())),
        (ValueError, lambda: gated_recurrence_grad(x, x, x, lam, x, grad_final_state=h[:1])),
        (TypeError, lambda: gated_recurrence_update(h.bfloat16(), x[:, 0], x[:, 0], x[:, 0], lam)),
        (ValueError, lambda: gated_recurrence_update(h[:1], x[:, 0], x[:, 0], x[:, 0], lam)),
        (ValueError, lambda: gated_recurrence_update(torch.zeros((8, 2), device="cuda").t(), x[:, 0], x[:, 0], x[:, 0], lam, inplace=True)),
    ]
    for k, (error, call) in enumerate(cases):
        with pytest.raises(error):
            call()
            pytest.fail(f"case {k} was not refused")


def test_c_refusals_need_no_gpu():
    """Arguments that the library has to refuse before it touches a device."""
    from mamba2_b200 import _lib
    lib = _lib.load()
    P, G, S = _lib.GatedRecurrenceParams, _lib.GatedRecurrenceGrads, _lib.GatedRecurrenceUpdateParams

    def params(**kw):
        p = P(2, 70, 8, 560, 8, 560, 8, 560, 8, 0, 8.0, 256, 256, 256, 256, None, None, 256, None, None, None)
        for k, v in kw.items():
            setattr(p, k, v)
        return p

    grads = G(560, 8, 256, None, 256, 256, 256, 256, None)
    assert lib.ssd_gated_recurrence(None, None) == 1
    bad = [dict(batch=0), dict(seqlen=0), dict(dim=-1), dict(dtype=2), dict(scale=-1.0), dict(scale=float("nan")),
           dict(scale=float("inf"))]
    for kw in bad + [dict(x=None), dict(decay=None), dict(y=None)]:
        assert lib.ssd_gated_recurrence(params(**kw), None) == 1, kw
        assert lib.ssd_last_error()
    assert lib.ssd_gated_recurrence(params(seqlen=1 << 31), None) == 2
    assert lib.ssd_gated_recurrence(params(batch=1 << 30, dim=1 << 20), None) == 2
    need = lib.ssd_gated_recurrence_grad_workspace_bytes(params())
    assert need > lib.ssd_gated_recurrence_grad_workspace_bytes(params(checkpoints=256)) > 0
    for kw in bad:
        assert lib.ssd_gated_recurrence_grad_workspace_bytes(params(**kw)) == 0, kw
        assert lib.ssd_gated_recurrence_grad(params(**kw), grads, 256, need, None) == 1, kw
    assert lib.ssd_gated_recurrence_grad(params(), None, 256, need, None) == 1
    assert lib.ssd_gated_recurrence_grad(params(), G(560, 8, None, None, 256, 256, 256, 256, None), 256, need, None) == 1
    assert lib.ssd_gated_recurrence_grad(params(), G(560, 8, 256, None, 256, None, 256, 256, None), 256, need, None) == 1
    assert lib.ssd_gated_recurrence_grad(params(), grads, 256, need - 1, None) == 4
    assert lib.ssd_gated_recurrence_grad(params(), grads, None, need, None) == 4
    assert lib.ssd_gated_recurrence_grad(params(), grads, 264, need, None) == 3
    good = (2, 8, 8, 8, 8, 0, 8.0, 256, 256, 256, 256, 256, 256, 256)
    for k, v in ((0, 0), (1, -1), (5, 3), (6, -1.0), (7, None), (10, None), (11, None), (12, None), (13, None)):
        p = S(*(v if j == k else a for j, a in enumerate(good)))
        assert lib.ssd_gated_recurrence_update(p, None) == 1, k
