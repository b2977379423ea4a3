"""Bounds of the float32 linear cross entropy, derived for what it computes with (two f16 terms per value, three
products per pair), and checks on the CPU that they tell it from one with a term missing.

A logit is off by at most
- 3 * 2^-22 of the 2-norm of its products, twice (roundings of the terms, and lo * lo; independent, so they add
  up like a random walk, with twice the room);
- 24 * 2^-23 of the largest partial sum within a segment of 128 products (the tensor cores' adds cut, and there
  are 3 products x 8 adds in a segment), 2^-24 of the sum per segment behind it.
Gradients, 2-norm: twice the largest logit error (dl moves by a factor of at most that), and the product's own
error c |dl| |M| with the c of test_lm_numerics.
"""
import math

import pytest
import torch

from mamba2_b200 import linear_cross_entropy, linear_cross_entropy_grad
from test_lm_numerics import grad_constant, ints, reference

SIZES = [(64, 513, 65), (127, 300, 40), (129, 700, 128), (200, 500, 200), (150, 131, 1000), (33, 1500, 24)]


def inputs(t, v, d):
    g = torch.Generator().manual_seed(t)
    w = torch.randn((v, d), generator=g) / math.sqrt(d)
    y = torch.randint(0, v, (t,), generator=g)
    x = torch.randn((t, d), generator=g) + 6.0 * torch.rand((t, 1), generator=g) * w[y]
    return x, w, y


def logit_bound(x, w):
    x, w = x.double(), w.double()
    worst = torch.zeros(len(x), len(w), dtype=torch.float64)
    total = torch.zeros_like(worst)
    for k0 in range(0, x.shape[1], 128):
        run = torch.cumsum(x[:, None, k0:k0 + 128] * w[None, :, k0:k0 + 128], 2)
        worst = torch.maximum(worst, run.abs().amax(2))
        total = total + run[..., -1]
    norm = ((x * x) @ (w * w).t()).sqrt()
    return float((6 * 2.0 ** -22 * norm + 24 * 2.0 ** -23 * worst + x.shape[1] / 128 * 2.0 ** -24 * total.abs()).max())


def bounds(x, w, y):
    """(largest logit error, relative bounds of both gradients, float64 loss and gradients)."""
    x, w = x.double(), w.double()
    e = logit_bound(x, w)
    loss, lse, dl, s = reference(x, w, y, torch.ones(len(y), dtype=torch.float64))
    out = []
    for a, m in ((dl, w), (dl.t(), x)):
        ref = a @ m
        own = grad_constant(a.shape[1], s) * float((a.abs() @ m.abs()).norm()) / float(ref.norm())
        out.append((ref, 2 * e + own))
    return e, loss, lse, out


def rel(got, ref):
    return float((got.double().cpu() - ref).norm() / ref.norm())


@pytest.mark.gpu
@pytest.mark.parametrize("t,v,d", SIZES)
def test_f32_loss_and_gradients(t, v, d):
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    x, w, y = inputs(t, v, d)
    e, loss, lse, grads = bounds(x, w, y)
    rows, l2 = linear_cross_entropy(x.cuda(), w.cuda(), y.cuda(), reduction="none", return_lse=True)
    room = 2 * e + 2.0 ** -21 + 4 * 2.0 ** -24 * (1 + loss + lse.abs())
    assert ((rows.double().cpu() - loss).abs() <= room).all() and ((l2.double().cpu() - lse).abs() <= room).all()
    _, dx, dw = linear_cross_entropy_grad(x.cuda(), w.cuda(), y.cuda(), reduction="sum")
    for got, (ref, bound) in zip((dx, dw), grads):
        assert rel(got, ref) <= bound, (rel(got, ref), bound)


def planes(m, terms):
    """Rows of m as `terms` f16 terms of their values times a power of two, as float64."""
    m = m.double()
    scale = 2.0 ** (14 - torch.floor(torch.log2(m.abs().amax(1, keepdim=True).clamp(min=1e-300))))
    hi = (m * scale).half().double()
    lo = (m * scale - hi).half().double() if terms == 2 else torch.zeros_like(hi)
    return hi / scale, lo / scale


def product(a, b, terms_a, terms_b):
    """a @ b^T from the planes of both."""
    (ah, al), (bh, bl) = planes(a, terms_a), planes(b, terms_b)
    return ah @ bh.t() + ah @ bl.t() + al @ bh.t()


@pytest.mark.parametrize("t,v,d", SIZES)
def test_the_bounds_see_missing_low_terms(t, v, d):
    """The same arithmetic in float64: with all terms inside the bounds, without a low term outside."""
    x, w, y = inputs(t, v, d)
    e, _, _, grads = bounds(x, w, y)
    for tx, tw in ((2, 2), (1, 1), (1, 2), (2, 1)):
        s = product(x, w, tx, tw)
        p = torch.softmax(s, 1)
        p[torch.arange(t), y] -= 1.0
        got = product(p, w.t().contiguous(), tx, tw), product(p.t().contiguous(), x.t().contiguous(), tx, tw)
        inside = [rel(a, ref) <= bound for a, (ref, bound) in zip(got, grads)]
        assert inside == [tx == tw == 2] * 2, (tx, tw, [(rel(a, r), b) for a, (r, b) in zip(got, grads)])


@pytest.mark.parametrize("long", ["hidden", "weight"])
def test_17_bit_values_see_a_missing_product(long):
    """The exact logits of test_lm_numerics.test_f32_values_of_17_bits, without the product of one low term."""
    x, w = ints((200, 64), 17, 0, 15), ints((300, 64), 2, 1, 1)
    if long == "weight":
        x, w = ints((200, 64), 2, 0, 1), ints((300, 64), 17, 1, 15)
    y = torch.randint(0, 300, (200,), generator=torch.Generator().manual_seed(2))
    loss, lse, _, s = reference(x, w, y, torch.ones(200, dtype=torch.float64))
    bound = 2.0 ** -21 + 2 * 2.0 ** -24 * s.abs().max() + 4 * 2.0 ** -24 * (1 + loss.abs() + lse.abs())
    for tx, tw in ((2, 2), (1, 2), (2, 1)):
        got = reference_loss(product(x, w, tx, tw), y)
        whole = tx == 2 if long == "hidden" else tw == 2
        assert bool(((got - loss).abs() <= bound).all()) == whole


def reference_loss(s, y):
    return torch.nn.functional.cross_entropy(s, y, reduction="none")
