"""The gated feed-forward block and its gradients: the CUDA kernels against plain float64 restatements, and their
refusals.

Tolerances.  u = 2^-24 and v = 2^-8 are the largest relative errors of a rounding to float32 and bfloat16.
- Products of bfloat16 values are exact in float32; the tensor cores' adds may truncate (2 u of the largest partial
  sum), and sums of segments are rounded: a product of K terms is off by at most 2 K u S, S the same product of the
  magnitudes.  Float32 operands are three bfloat16 terms; what is left out is below 3 * 2^-24 of each product: (2 K + 6) u S.
  A second or third term below bfloat16's smallest normal number 2^-126 counts as zero: an operand is off by up to
  2 * 2^-126 more, which 2^-125 (sum|a| + sum|b|) takes in (it matters below 2^-110: rows times 2^-60 twice).
- With s the largest error of g and u over their magnitudes' products, act and act' (slopes below 1.13, second
  derivatives below 0.8, own arithmetic 32 u) move h = act(g) u by at most
  e_h = (1.13 |u| + |act(g)|) s + 32 u |h|, dg and du alike by e_g = |dh| (1.13 s |u| + 1.13 s) + ..., all
  evaluated with 2 for these factors; h, dg and du are rounded to bfloat16: v of themselves.
- A result is off by the product of its operands' errors' magnitudes with the other operand, its own product's
  error, and its rounding.
These are worst cases, element by element.  Beside them 2-norms: each independent rounding to bfloat16 has a relative standard
deviation of at most v / sqrt(3) / 2 (uniform over half a step either side, values spread over an octave), so two in a row (operand and
result) give at most v * 0.6: the bound is v.  Float32: 3e-6.
relu's slope jumps: a g within its error of zero may go either way, so relu is compared where |g| > s only through inputs
that leave no such g (they are checked to).
"""
import math

import pytest
import torch

from mamba2_b200 import gated_feed_forward, gated_feed_forward_grad

gpu = pytest.mark.gpu
U, V = 2.0 ** -24, 2.0 ** -8
DT = {"f32": torch.float32, "bf16": torch.bfloat16}
ACTS = ("silu", "gelu", "gelu_tanh", "relu")


@pytest.fixture(autouse=True)
def _need_gpu(request):
    if request.node.get_closest_marker("gpu") and not torch.cuda.is_available():
        pytest.skip("no CUDA device")


def act64(g, name):
    if name == "relu":
        return torch.clamp(g, min=0), (g > 0).double()
    if name == "silu":
        s = torch.sigmoid(g)
        return g * s, s * (1 + g * (1 - s))
    if name == "gelu":
        p = 0.5 * torch.erfc(-g / math.sqrt(2))
        return g * p, p + g * torch.exp(-0.5 * g * g) / math.sqrt(2 * math.pi)
    c = math.sqrt(2 / math.pi)
    t = torch.tanh(c * (g + 0.044715 * g ** 3))
    return 0.5 * g * (1 + t), 0.5 * (1 + t) + 0.5 * g * (1 - t * t) * c * (1 + 3 * 0.044715 * g * g)


def inputs(t, d, f, o, dtype, seed=0):
    gen = torch.Generator().manual_seed(seed)

    def rnd(*shape, scale=1.0):
        return (torch.randn(shape, generator=gen) * scale).to(DT[dtype])

    return (rnd(t, d), rnd(f, d, scale=1 / math.sqrt(d)), rnd(f, d, scale=1 / math.sqrt(d)), rnd(o, f, scale=1 / math.sqrt(f)),
            rnd(t, o))


def reference(x, wg, wu, wd, dy, act, dtype):
    """(y, gradients) in float64 and a bound for each value."""
    x, wg, wu, wd, dy = (t.double() for t in (x, wg, wu, wd, dy))
    k = 2 if dtype == "bf16" else 2
    extra = 0 if dtype == "bf16" else 6
    round_op = V if dtype == "bf16" else 3 * U   # operands made on the way

    def prod(a, b, ea=None, eb=None):
        """a @ b and its error's bound, given those of a and b."""
        s = a.abs() @ b.abs()
        e = (k * a.shape[1] + extra) * U * s
        if dtype == "f32":
            e = e + 2.0 ** -125 * (a.abs().sum(1)[:, None] + b.abs().sum(0)[None])
        if ea is not None:
            e = e + ea @ b.abs()
        if eb is not None:
            e = e + a.abs() @ eb
        return a @ b, e

    g, sg = prod(x, wg.t())
    u, su = prod(x, wu.t())
    v, dv = act64(g, act)
    h = v * u
    eh = 1.2 * sg * u.abs() + su * v.abs() + 2 * sg * su + 32 * U * h.abs()
    eh = eh + round_op * (h.abs() + eh)
    out_round = V if dtype == "bf16" else 2 * U
    y, ey = prod(h, wd.t(), ea=eh)
    dh, edh = prod(dy, wd)
    dg, du = dh * u * dv, dh * v
    edg = edh * (u * dv).abs() + dh.abs() * (su * dv.abs() + u.abs() * 0.9 * sg) + 2 * edh * su + 64 * U * dg.abs() + 32 * U * (dh * u).abs()
    edu = edh * v.abs() + dh.abs() * 1.2 * sg + 2 * edh * sg + 32 * U * du.abs()
    edg, edu = edg + round_op * (dg.abs() + edg), edu + round_op * (du.abs() + edu)
    a, ea = prod(dg, wg, ea=edg)
    b, eb = prod(du, wu, ea=edu)
    dx, edx = a + b, ea + eb + 2 * U * (a.abs() + b.abs()) + (k * dg.shape[1]) * U * ((dg.abs() @ wg.abs()) + (du.abs() @ wu.abs()))
    res = [(y, ey), (dx, edx), prod(dg.t(), x, ea=edg.t()), prod(du.t(), x, ea=edu.t()), prod(dy.t(), h, eb=eh)]
    near = float((g.abs() - sg).min())
    return [(r, e + out_round * (r.abs() + e) + 1e-38) for r, e in res], near


def close(got, ref, bound, dtype):
    got = got.double().cpu()
    assert torch.isfinite(got).all()
    worst = float(((got - ref).abs() - bound).max())
    assert worst <= 0, worst
    if ref.numel() >= 64:
        rel = float((got - ref).norm() / ref.norm())
        assert rel <= (V if dtype == "bf16" else 3e-6), rel


def separated(t, d, f, o, dtype, act, seed):
    """Inputs, of the first seeds, whose gates are all clear of zero where relu needs it."""
    for s in range(seed, seed + 200):
        ins = inputs(t, d, f, o, dtype, s)
        refs, near = reference(*ins, act, dtype)
        if act != "relu" or near > 0:
            return ins, refs
    raise AssertionError("no such inputs")


SHAPES = [(1, 1, 1, 1), (1, 64, 64, 64), (2, 100, 33, 7), (3, 65, 130, 9), (5, 256, 96, 40), (8, 72, 257, 65), (9, 64, 64, 64),
          (33, 7, 5, 3), (64, 200, 127, 129), (127, 65, 128, 64), (128, 128, 129, 256), (129, 130, 200, 72), (200, 320, 300, 100),
          (257, 64, 64, 300), (300, 1000, 64, 64)]


@gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("t,d,f,o", SHAPES)
def test_forward_and_gradients(t, d, f, o, dtype):
    ins, refs = separated(t, d, f, o, dtype, "silu", t + d)
    c = [a.cuda() for a in ins]
    y = gated_feed_forward(*c[:4], check_status=True)
    assert y.dtype == DT[dtype] and y.shape == (t, o)
    close(y, *refs[0], dtype)
    grads = gated_feed_forward_grad(*c, check_status=True)
    for g, (ref, bound) in zip(grads, refs[1:]):
        assert g.dtype == DT[dtype] and g.shape == ref.shape
        close(g, ref, bound, dtype)


@gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("t", [3, 50, 150])
def test_activations(t, act, dtype):
    ins, refs = separated(t, 40, 24, 16, dtype, act, 7 * t)
    c = [a.cuda() for a in ins]
    close(gated_feed_forward(*c[:4], activation=act), *refs[0], dtype)
    for g, (ref, bound) in zip(gated_feed_forward_grad(*c, activation=act), refs[1:]):
        close(g, ref, bound, dtype)


@gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("t", [2, 200])
def test_gates_of_any_size(t, act, dtype):
    """g from 2^3 to 2^100 (its square is beyond float32) either way, u = 1: act(g) is g or 0 and its slope 1 or 0, up to
    (1 + |g|) e^-|g| (silu; the others are nearer)."""
    size = torch.tensor([2.0 ** 70, 2.0 ** 100]) if t == 2 else 2.0 ** torch.arange(3, 101).repeat(3)[:t].float()
    tail = ((1 + size.double()) * torch.exp(-size.double()) * 1.001 + 1e-30)[:, None]
    for sign in (1.0, -1.0):
        x = torch.stack([sign * size, torch.ones(t)], 1).to(DT[dtype]).cuda()
        wg, wu, wd = (torch.tensor([row], device="cuda").to(DT[dtype]) for row in ([1.0, 0.0], [0.0, 1.0], [1.0]))
        dy = torch.ones((t, 1), dtype=DT[dtype], device="cuda")
        y = gated_feed_forward(x, wg, wu, wd, activation=act).double().cpu()
        dx = gated_feed_forward_grad(x, wg, wu, wd, dy, activation=act)[0].double().cpu()
        on = 1.0 if sign > 0 else 0.0
        for got, want in ((y, on * size.double()[:, None]), (dx, on * torch.stack([torch.ones(t), size], 1).double())):
            assert torch.isfinite(got).all()
            assert float(((got - want).abs() - (V * want + tail)).max()) <= 0


@gpu
@pytest.mark.parametrize("dtype,wd", [("bf16", torch.float32), ("f32", torch.bfloat16)])
def test_weight_grad_dtype(dtype, wd):
    ins, refs = separated(140, 96, 72, 64, dtype, "silu", 3)
    c = [a.cuda() for a in ins]
    want = gated_feed_forward_grad(*c)
    got = gated_feed_forward_grad(*c, weight_grad_dtype=wd)
    assert torch.equal(got[0], want[0])
    for g, w in zip(got[1:], want[1:]):
        assert g.dtype == wd
        if wd is torch.float32:     # the same sums, not rounded
            assert torch.equal(g.to(torch.bfloat16), w)
        else:
            assert torch.equal(g, w.to(torch.bfloat16))


@gpu
def test_what_is_not_needed_is_none():
    c = [a.cuda() for a in inputs(140, 96, 72, 64, "bf16", 4)]
    want = gated_feed_forward_grad(*c)
    only = gated_feed_forward_grad(*c, need_weight_grad=False)
    assert torch.equal(only[0], want[0]) and only[1:] == (None, None, None)
    only = gated_feed_forward_grad(*c, need_input_grad=False)
    assert only[0] is None and all(torch.equal(p, q) for p, q in zip(only[1:], want[1:]))
    assert gated_feed_forward_grad(*c, need_input_grad=False, need_weight_grad=False) == (None,) * 4


def grad_params(c, **kw):
    """The C call's structs for x, w_gate, w_up, w_down, grad_y and the gradients' tensors that are wanted."""
    from mamba2_b200 import _lib
    x, wg, wu, wd, dy = c
    (t, d), (f, _), o = x.shape, wg.shape, wd.shape[0]
    code = int(x.dtype == torch.bfloat16)
    p = _lib.GatedFfParams(t, d, f, o, d, d, d, f, code, 0, *(a.data_ptr() for a in (x, wg, wu, wd)), None)
    ptr = [None if kw.get(n) is None else kw[n].data_ptr() for n in ("grad_x", "grad_w_gate", "grad_w_up", "grad_w_down")]
    return p, _lib.GatedFfGrads(o, dy.data_ptr(), *ptr, code, 0)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_what_is_not_needed_takes_no_workspace(dtype):
    """h is there for w_down's gradient alone, dg, du and dh are for the others."""
    from mamba2_b200 import _lib
    size = _lib.load().ssd_gated_ff_grad_workspace_bytes
    c = [torch.empty(s, dtype=DT[dtype]) for s in ((1000, 64), (128, 64), (128, 64), (64, 128), (1000, 64))]
    g = dict(zip(("grad_x", "grad_w_gate", "grad_w_up", "grad_w_down"), c))
    plane = 1000 * 128 * 2 * (3 if dtype == "f32" else 1)
    need = {k: size(*grad_params(c, **{n: g[n] for n in names})) for k, names in dict(
        all=list(g), x=["grad_x"], in_=["grad_w_gate", "grad_w_up"], down=["grad_w_down"]).items()}
    assert need["all"] - need["x"] >= plane and need["all"] - need["in_"] >= plane
    assert need["all"] - need["down"] >= 2 * plane + 1000 * 128 * 4


@gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("t,d,f,o", [(3, 40, 24, 16), (140, 96, 72, 64), (300, 65, 130, 9)])
def test_each_gradient_alone(t, d, f, o, dtype):
    """Through the C entry point, which takes any of them; workspaces full of NaN; the status word is cleared in any case."""
    from mamba2_b200 import _lib
    lib = _lib.load()
    ins, refs = separated(t, d, f, o, dtype, "silu", 20)
    c = [a.cuda() for a in ins]
    names = ("grad_x", "grad_w_gate", "grad_w_up", "grad_w_down")
    full = dict(zip(names, gated_feed_forward_grad(*c)))
    ref = dict(zip(names, refs[1:]))
    for wanted in (("grad_x",), ("grad_w_gate", "grad_w_up"), ("grad_w_down",), ("grad_x", "grad_w_down"), ()):
        out = {n: torch.full_like(full[n], float("nan")) for n in wanted}
        p, g = grad_params(c, **out)
        ws = torch.full((max(lib.ssd_gated_ff_grad_workspace_bytes(p, g), 256),), 255, dtype=torch.uint8, device="cuda")
        _lib.check(lib.ssd_gated_ff_grad(p, g, ws.data_ptr(), ws.numel(), torch.cuda.current_stream().cuda_stream))
        _lib.check_device_status(ws)
        for n in wanted:
            close(out[n], *ref[n], dtype)
            if n != "grad_w_down":
                assert torch.equal(out[n], full[n]), n


@gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("t", [2, 7, 40, 150])
def test_strides(t, dtype):
    """Weights that are row or column slices of a larger one, batches with a stride, transposes."""
    d, f, o = 48, 40, 56
    g = torch.Generator().manual_seed(t)
    fused = (torch.randn((2 * f + 3, d + 5), generator=g) / math.sqrt(d)).to(DT[dtype]).cuda()
    big = torch.randn((t, d + o + 11), generator=g).to(DT[dtype]).cuda()
    down = (torch.randn((f, o), generator=g) / math.sqrt(f)).to(DT[dtype]).cuda().t()
    for at in (0, 1, 5):
        x, dy = big[:, at:at + d], big[:, d + at:d + at + o]
        wg, wu = fused[:f, at:at + d], fused[f + 3:, at:at + d]
        plain = [a.contiguous() for a in (x, wg, wu, down, dy)]
        refs, _ = reference(*(a.cpu() for a in plain), "silu", dtype)
        close(gated_feed_forward(x, wg, wu, down), *refs[0], dtype)
        for got, (ref, bound) in zip(gated_feed_forward_grad(x, wg, wu, down, dy), refs[1:]):
            close(got, ref, bound, dtype)
    batch = plain[0][None].expand(3, t, d)
    y = gated_feed_forward(batch, *plain[1:4])
    assert y.shape == (3, t, o) and torch.equal(y[0], y[2])


@gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("t", [1, 3, 9])
def test_rows_that_start_anywhere(t, dtype):
    """Few tokens: views of buffers that hold NaN around them, at every start of a row within 16 bytes; rows of several steps of a warp."""
    d, f, o = 777, 251, 21
    ins = inputs(t, d, f, o, dtype, 3)
    refs, _ = reference(*ins, "silu", dtype)
    for at in range(9):
        views = []
        for k, a in enumerate(ins[:4]):
            wide = torch.full((a.shape[0], a.shape[1] + 16 + k), float("nan"), dtype=DT[dtype], device="cuda")
            view = wide[:, (at + 3 * k) % 9:][:, :a.shape[1]]
            view.copy_(a)
            views.append(view)
        close(gated_feed_forward(*views), *refs[0], dtype)


@gpu
@pytest.mark.parametrize("t", [5, 8, 9, 16, 17, 24, 25])
def test_float32_slices_of_wider_rows(t):
    """Rows of a few tokens and of weights at one distance, a multiple of 16 bytes, whose first starts off 16 bytes: passes of 8 tokens, whole
    and cut off, and what takes over behind them.  NaN lies around the views."""
    d, f, o = 777, 251, 21
    ins = inputs(t, d, f, o, "f32", 19)
    refs, _ = reference(*ins, "silu", "f32")
    for at in ((0, 0, 0, 0), (1, 0, 0, 0), (0, 1, 2, 0), (0, 2, 0, 3), (0, 0, 0, 1), (3, 2, 1, 2)):
        views = []
        for a, start in zip(ins[:4], at):
            wide = torch.full((a.shape[0], (a.shape[1] + 7) // 4 * 4), float("nan"), device="cuda")
            view = wide[:, start:start + a.shape[1]]
            view.copy_(a)
            views.append(view)
        close(gated_feed_forward(*views), *refs[0], "f32")


def test_which_form_takes_few_tokens():
    """The limits go by sizes and by where rows start, base addresses among it; seen by the workspace, which then holds the hidden values alone."""
    from mamba2_b200 import _lib
    lib = _lib.load()

    def few(tokens, dtype=0, dim=2560, hidden=7680, **kw):
        p = _lib.GatedFfParams(tokens, dim, hidden, dim, dim, dim, dim, hidden, dtype, 0, 256, 256, 256, 256, 256)
        for k, v in kw.items():
            setattr(p, k, v)
        size = lib.ssd_gated_ff_workspace_bytes(p)
        only = 256 + (tokens * ((hidden + 7) // 8 * 8) * 4 + 255) // 256 * 256
        assert size >= only
        return size == only

    def limit(**kw):
        most = max(t for t in range(1, 40) if few(t, **kw))
        assert all(few(t, **kw) == (t <= most) for t in range(1, 40))
        return most

    assert limit(dtype=1) == 4 and limit(dtype=1, x=258) == 4
    assert limit() == 24 and limit(w_down=260) == 24 and limit(w_down_stride_row=7681) == 24
    assert limit(w_gate=260) == 16 and limit(w_up=264) == 16 and limit(w_up_stride_row=2561) == 16
    assert limit(x=260) == 8 and limit(x_stride_row=2562) == 8 and limit(x=260, w_gate=260) == 8
    assert limit(dim=2559, x_stride_row=2560, w_gate_stride_row=2560, w_up_stride_row=2560) == 16
    assert limit(hidden=7681, w_down_stride_row=7684) == 24
    small, large = dict(dim=768, hidden=2048), dict(dim=4096, hidden=12288)
    assert limit(**small, w_up=260) == 24 and limit(**small, x=260) == 16 and limit(**large) == 24 and limit(**large, w_down=260) == 16


@gpu
@pytest.mark.parametrize("act", ["silu", "relu"])
@pytest.mark.parametrize("t,d,f,o", [(1, 40, 7, 64), (2, 24, 9, 130), (3, 40, 16, 65), (4, 33, 24, 128), (4, 8, 5, 200)])
def test_few_tokens_round_once(t, d, f, o, act):
    """bfloat16, few tokens: the products run in float32, so the results' own rounding is the only one to bfloat16.  The bound is the
    one above without v for h.  (Few hidden values, so that float32's worst case is small beside what a rounded h would do.)"""
    ins = inputs(t, d, f, o, "bf16", 18)
    x, wg, wu, wd = (a.double() for a in ins[:4])
    sg, su = (2 * d * U * (x.abs() @ w.abs().t()) for w in (wg, wu))
    g, u = x @ wg.t(), x @ wu.t()
    v, _ = act64(g, act)
    h = v * u
    eh = 1.2 * sg * u.abs() + su * v.abs() + 2 * sg * su + 33 * U * h.abs()
    y, e = h @ wd.t(), 2 * f * U * (h.abs() @ wd.abs().t()) + eh @ wd.abs().t()
    close(gated_feed_forward(*(a.cuda() for a in ins[:4]), activation=act), y, e + V * (y.abs() + e) + 1e-38, "bf16")


@gpu
@pytest.mark.parametrize("t,d,f,o", [(300, 4096, 64, 64), (64, 64, 4096, 64), (1000, 64, 64, 64), (16, 8, 2000, 8), (5000, 24, 16, 8)])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_long_reductions(t, d, f, o, dtype):
    """Few tiles and long K ranges: the ranges are split."""
    ins = inputs(t, d, f, o, dtype, 5)
    refs, _ = reference(*ins, "silu", dtype)
    c = [a.cuda() for a in ins]
    close(gated_feed_forward(*c[:4]), *refs[0], dtype)
    for g, (ref, bound) in zip(gated_feed_forward_grad(*c), refs[1:]):
        close(g, ref, bound, dtype)


@gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_large_and_small_values(dtype):
    """Rows, columns and weights of very different sizes; float32 keeps its digits down to 2^-110."""
    t, d, f, o = 150, 64, 64, 64
    x, wg, wu, wd, dy = inputs(t, d, f, o, dtype, 6)
    x[3] *= 2.0 ** 40
    x[5] *= 2.0 ** -60
    wu[7] *= 2.0 ** 30
    wd[9] *= 2.0 ** -50
    wd[:, 11] *= 2.0 ** 20
    dy[13] *= 2.0 ** -70
    refs, _ = reference(x, wg, wu, wd, dy, "silu", dtype)
    c = [a.cuda() for a in (x, wg, wu, wd, dy)]
    ys = gated_feed_forward(*c[:4]).double().cpu()
    assert float(((ys - refs[0][0]).abs() - refs[0][1]).max()) <= 0
    for g, (ref, bound) in zip(gated_feed_forward_grad(*c), refs[1:]):
        assert float(((g.double().cpu() - ref).abs() - bound).max()) <= 0


@gpu
def test_values_that_are_not_finite_stay_in_their_rows():
    for dtype in ("f32", "bf16"):
        for t in (6, 150):
            c = [a.cuda() for a in inputs(t, 64, 64, 64, dtype, 8)]
            y0, g0 = gated_feed_forward(*c[:4]), gated_feed_forward_grad(*c)
            for bad in (float("nan"), float("inf")):
                x = c[0].clone()
                x[2, 5] = bad
                y = gated_feed_forward(x, *c[1:4])
                keep = torch.arange(t, device="cuda") != 2
                assert torch.equal(y[keep], y0[keep]) and not torch.isfinite(y[2]).all()
                assert torch.equal(gated_feed_forward_grad(x, *c[1:])[0][keep], g0[0][keep])


@gpu
@pytest.mark.parametrize("dtype,t", [("f32", 6), ("bf16", 3), ("bf16", 150), ("f32", 150)])
def test_what_becomes_of_an_infinity(dtype, t):
    """Where the formula keeps one (nothing negative meets it) it stays one, but for float32 operands in three terms: what is left of it for
    the second is NaN."""
    x, w = torch.ones((t, 64)), torch.full((64, 64), 0.125)
    x[2, 5] = math.inf
    x, w = x.to(DT[dtype]).cuda(), w.to(DT[dtype]).cuda()
    y = gated_feed_forward(x, w, w, w)
    assert (torch.isnan(y[2]) if (dtype, t) == ("f32", 150) else torch.isposinf(y[2])).all()
    keep = torch.arange(t, device="cuda") != 2
    assert torch.isfinite(y[keep]).all()


@gpu
def test_large_tiles_against_float64():
    """Several tiles each way, ragged, on the GPU's own float64."""
    for dtype, (t, d, f, o) in (("bf16", (1500, 1024, 1400, 900)), ("f32", (700, 500, 600, 300))):
        ins = [a.cuda() for a in inputs(t, d, f, o, dtype, 9)]
        x, wg, wu, wd, dy = (a.double().requires_grad_() for a in ins)
        y = (torch.nn.functional.silu(x @ wg.t()) * (x @ wu.t())) @ wd.t()
        refs = torch.autograd.grad(y, (x, wg, wu, wd), dy)
        got = (gated_feed_forward(*ins[:4]),) + gated_feed_forward_grad(*ins)
        for g, ref in zip(got, (y.detach(),) + refs):
            rel = float((g.double() - ref).norm() / ref.norm())
            assert rel <= (V if dtype == "bf16" else 3e-6), rel


@gpu
@pytest.mark.parametrize("act", ["silu", "gelu", "gelu_tanh"])
def test_gradients_against_differences(act):
    """Central differences of the float64 block along a random direction of every input."""
    ins = inputs(40, 24, 20, 16, "f32", 10)
    got = [g.double().cpu() for g in gated_feed_forward_grad(*(a.cuda() for a in ins), activation=act)]
    base = [a.double() for a in ins]

    def value(ts):
        x, wg, wu, wd = ts
        return float(((act64(x @ wg.t(), act)[0] * (x @ wu.t())) @ wd.t() * base[4]).sum())

    gen = torch.Generator().manual_seed(11)
    for k in range(4):
        v = torch.randn(base[k].shape, generator=gen, dtype=torch.float64)
        hi, lo = list(base[:4]), list(base[:4])
        hi[k], lo[k] = base[k] + 1e-5 * v, base[k] - 1e-5 * v
        want = (value(hi) - value(lo)) / 2e-5
        assert abs(float((got[k] * v).sum()) - want) <= 1e-5 * float((got[k] * v).abs().sum()) + 1e-6


@gpu
def test_equal_calls_give_equal_bits_and_graphs_replay():
    c = [a.cuda() for a in inputs(300, 256, 320, 256, "bf16", 12)]
    few = [c[0][:3], *c[1:4]]

    def step():
        return (gated_feed_forward(*c[:4]), gated_feed_forward(*few)) + gated_feed_forward_grad(*c)

    want = step()
    assert all(torch.equal(p, q) for p, q in zip(step(), want))
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    torch.cuda.current_stream().wait_stream(s)
    graphs = []
    for _ in range(2):
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
    for t in c:
        t.copy_(torch.randn_like(t, dtype=torch.float32) * 0.1)
    graphs[1][0].replay()
    fresh = step()
    torch.cuda.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(graphs[1][1], fresh))


@gpu
def test_two_streams_at_once():
    sets = [[a.cuda() for a in inputs(500, 300, 400, 200, "bf16", s)] for s in (13, 14)]
    want = [gated_feed_forward_grad(*t) for t in sets]
    streams = [torch.cuda.Stream() for _ in sets]
    torch.cuda.synchronize()
    got = [None, None]
    for _ in range(3):
        for k, (s, t) in enumerate(zip(streams, sets)):
            with torch.cuda.stream(s):
                got[k] = gated_feed_forward_grad(*t)
    torch.cuda.synchronize()
    for p, q in zip(got, want):
        assert all(torch.equal(a, b) for a, b in zip(p, q))


@gpu
def test_weights_just_written():
    """Kernels of the call that are set up early must not read what the kernel before is still writing."""
    c = [a.cuda() for a in inputs(2, 512, 4096, 512, "bf16", 15)]
    for t in (2, 200):
        x = torch.randn((t, 512), device="cuda").to(torch.bfloat16)
        for k in range(20):
            new = [torch.full_like(w, 0.001 * (k + 1)) for w in c[1:4]]
            torch.cuda.synchronize()
            want = gated_feed_forward(x, *new)
            torch.cuda.synchronize()
            for w in c[1:4]:
                w.fill_(-7.0)
            for w, n in zip(c[1:4], new):
                w.copy_(n)
            got = gated_feed_forward(x, *c[1:4])
            assert torch.equal(got, want)


@gpu
def test_empty():
    w = torch.ones((8, 4), device="cuda")
    d = torch.ones((6, 8), device="cuda")
    x = torch.zeros((2, 0, 4), device="cuda")
    assert gated_feed_forward(x, w, w, d).shape == (2, 0, 6)
    g = gated_feed_forward_grad(x, w, w, d, torch.zeros((2, 0, 6), device="cuda"))
    assert g[0].shape == x.shape and all(float(t.abs().max()) == 0 for t in g[1:])


@gpu
@pytest.mark.slow
def test_past_32_bit_offsets():
    """More than 2^31 hidden values: the last rows equal those of a short call."""
    t, d, f, o = 270_000, 64, 8192, 64
    gen = torch.Generator(device="cuda").manual_seed(16)
    x = torch.randn((t, d), generator=gen, device="cuda").to(torch.bfloat16)
    wg, wu = (torch.randn((f, d), generator=gen, device="cuda").mul_(0.125).to(torch.bfloat16) for _ in range(2))
    wd = torch.randn((o, f), generator=gen, device="cuda").mul_(0.01).to(torch.bfloat16)
    y = gated_feed_forward(x, wg, wu, wd)
    tail = gated_feed_forward(x[-256:], wg, wu, wd)
    assert float((y[-256:].float() - tail.float()).norm() / tail.float().norm()) <= V
    gx = gated_feed_forward_grad(x, wg, wu, wd, x, need_weight_grad=False)[0]
    short = gated_feed_forward_grad(x[-256:], wg, wu, wd, x[-256:], need_weight_grad=False)[0]
    assert float((gx[-256:].float() - short.float()).norm() / short.float().norm()) <= V


def test_refusals_need_no_gpu():
    x, w, d = torch.zeros((2, 4)), torch.zeros((8, 4)), torch.zeros((6, 8))
    with pytest.raises(ValueError, match="CUDA"):
        gated_feed_forward(x, w, w, d)
    with pytest.raises(ValueError, match="CUDA"):
        gated_feed_forward_grad(x, w, w, d, torch.zeros((2, 6)))
    with pytest.raises(TypeError, match="torch.Tensor"):
        gated_feed_forward(x.numpy(), w, w, d)


@gpu
def test_refusals():
    x, w, d = (torch.zeros(s, device="cuda") for s in ((2, 4), (8, 4), (6, 8)))
    dy = torch.zeros((2, 6), device="cuda")
    cases = [
        (ValueError, lambda: gated_feed_forward(x[:, :3], w, w, d)),
        (ValueError, lambda: gated_feed_forward(x, w, w[:4], d)),
        (ValueError, lambda: gated_feed_forward(x, w, w, d[:, :4])),
        (ValueError, lambda: gated_feed_forward(x, w[0], w[0], d)),
        (ValueError, lambda: gated_feed_forward(x, w, w, d.cpu())),
        (TypeError, lambda: gated_feed_forward(x, w.bfloat16(), w, d)),
        (TypeError, lambda: gated_feed_forward(x.half(), w.half(), w.half(), d.half())),
        (ValueError, lambda: gated_feed_forward(x, w, w, d, activation="tanh")),
        (ValueError, lambda: gated_feed_forward(x, w[:0], w[:0], d[:, :0])),
        (ValueError, lambda: gated_feed_forward_grad(x, w, w, d, dy[:1])),
        (TypeError, lambda: gated_feed_forward_grad(x, w, w, d, dy.bfloat16())),
        (ValueError, lambda: gated_feed_forward_grad(x, w, w, d, dy, weight_grad_dtype=torch.float16)),
    ]
    for k, (error, call) in enumerate(cases):
        with pytest.raises(error):
            call()
            pytest.fail(f"case {k} was not refused")


def test_c_refusals_need_no_gpu():
    """Arguments that the library has to refuse before it touches a device."""
    from mamba2_b200 import _lib
    lib = _lib.load()

    def params(**kw):
        p = _lib.GatedFfParams(50, 64, 96, 32, 64, 64, 64, 96, 1, 0, 256, 256, 256, 256, 256)
        for k, v in kw.items():
            setattr(p, k, v)
        return p

    def grads(**kw):
        g = _lib.GatedFfGrads(32, 256, 256, 256, 256, 256, 1, 0)
        for k, v in kw.items():
            setattr(g, k, v)
        return g

    bad = [dict(tokens=0), dict(dim=-1), dict(hidden=0), dict(dim_out=0), dict(dtype=2), dict(activation=4),
           dict(activation=-1), dict(x_stride_row=63), dict(w_gate_stride_row=63), dict(w_up_stride_row=0),
           dict(w_down_stride_row=95), dict(x=None), dict(w_gate=None), dict(w_up=None), dict(w_down=None)]
    assert lib.ssd_gated_ff(None, 256, 1 << 30, None) == 1
    for kw in bad:
        assert lib.ssd_gated_ff_workspace_bytes(params(**kw)) == 0, kw
        assert lib.ssd_gated_ff(params(**kw), 256, 1 << 30, None) == 1, kw
        assert lib.ssd_gated_ff_grad_workspace_bytes(params(**kw), grads()) == 0, kw
        assert lib.ssd_gated_ff_grad(params(**kw), grads(), 256, 1 << 30, None) == 1, kw
    assert lib.ssd_gated_ff(params(y=None), 256, 1 << 30, None) == 1
    assert lib.ssd_gated_ff(params(tokens=1 << 31), 256, 1 << 60, None) == 2
    for kw in (dict(grad_y=None), dict(grad_y_stride_row=31), dict(grad_weight_dtype=2), dict(grad_w_up=None)):
        assert lib.ssd_gated_ff_grad(params(), grads(**kw), 256, 1 << 30, None) == 1, kw
    assert lib.ssd_gated_ff_grad(params(), None, 256, 1 << 30, None) == 1
    need = lib.ssd_gated_ff_grad_workspace_bytes(params(), grads())
    assert need > lib.ssd_gated_ff_workspace_bytes(params()) > 256
    assert lib.ssd_gated_ff_grad(params(), grads(), 256, need - 1, None) == 4
    assert lib.ssd_gated_ff_grad(params(), grads(), None, need, None) == 4
    assert lib.ssd_gated_ff_grad(params(), grads(), 264, need, None) == 3
