"""The example that runs the language-model operators together around frozen mixer layers: the
loss falls, and its gradients are those of differences of the whole path."""
import math
import os
import sys

import pytest
import torch

pytestmark = pytest.mark.gpu
sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples"))


@pytest.fixture(autouse=True)
def _need_gpu():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")


def test_example_learns():
    import adapt_lm_ends
    losses, held_out, out = adapt_lm_ends.main(steps=12, vocab=67, d_model=256, n_layers=1, rows=2, length=160,
                                               verbose=False)
    losses = losses.cpu()
    assert torch.isfinite(losses).all() and torch.isfinite(held_out)
    assert float(losses[-3:].mean()) < float(losses[:2].mean()) - 0.3
    assert out.shape == (2, 8) and int(out.min()) >= 0 and int(out.max()) < 67


def test_path_gradients_against_differences():
    """loss(E, W) = CE(scale E[ids] + f, W) in float64 along random directions of E and W, against the
    kernels' float32 gradients: central differences, h^2 error below 1e-6 of the slope here."""
    from mamba2_b200 import embedding, embedding_grad, linear_cross_entropy_grad
    g = torch.Generator().manual_seed(1)
    vocab, dim, n, scale = 150, 32, 64, 3.0
    E, W = (torch.randn((vocab, dim), generator=g) / math.sqrt(dim) for _ in range(2))
    f = torch.randn((n, dim), generator=g)
    ids, y = torch.randint(0, vocab, (2, n), generator=g)
    y[::5] = -100
    h = embedding(ids.cuda(), E.cuda(), scale=scale) + f.cuda()
    loss, dh, dW = linear_cross_entropy_grad(h, W.cuda(), y.cuda())
    dE = embedding_grad(ids.cuda(), dh, vocab, scale=scale)

    def value(s, a, b):
        logits = (scale * (E.double() + s * a)[ids] + f.double()) @ (W.double() + s * b).t()
        return float(torch.nn.functional.cross_entropy(logits, y, ignore_index=-100))

    for seed in (2, 3):
        gd = torch.Generator().manual_seed(seed)
        a, b = (torch.randn((vocab, dim), generator=gd).double() for _ in range(2))
        num = (value(1e-4, a, b) - value(-1e-4, a, b)) / 2e-4
        parts = torch.cat([(dE.double().cpu() * a).flatten(), (dW.double().cpu() * b).flatten()])
        assert abs(num - float(parts.sum())) <= 1e-4 * float(parts.norm()) * math.sqrt(2)
