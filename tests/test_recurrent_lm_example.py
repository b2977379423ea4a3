"""The example that runs the block operators together with the language-model ends: that it runs, its gradients against
autograd of the same model in float64, and its single-token steps against its forward pass.

Tolerance of the float32 gradients: each operator's results are within 3e-6 (2-norm) of its formula's, and the
projections between them (float32 library products of 32 terms) within 2e-6; a gradient passes through at
most 2 layers x 4 of them each way, whose errors add up at worst: 16 x 5e-6 = 8e-5, times the at most
5-fold growth of a perturbation along two layers of this size: 4e-4.
"""
import math
import os
import sys

import pytest
import torch

from mamba2_b200 import gated_recurrence

pytestmark = pytest.mark.gpu
sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples"))


@pytest.fixture(autouse=True)
def _need_gpu():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")


def reference_loss(p, ids, targets, seq, layers):
    """The whole model in float64, token by token."""
    dim = p["table"].shape[1]
    h = math.sqrt(dim) * p["table"][ids]
    for k in range(layers):
        v, r, i = (h @ p[f"{k}.{n}"].t() for n in ("v", "r", "i"))
        la = -8.0 * torch.nn.functional.softplus(p[f"{k}.decay"]) * torch.sigmoid(r)
        b = torch.sqrt(-torch.expm1(2 * la)) * torch.sigmoid(i) * v
        state, ys = torch.zeros_like(h[:, 0]), []
        for t in range(ids.shape[1]):
            if t:
                state = state * (seq[:, t] == seq[:, t - 1])[:, None]
            state = torch.exp(la[:, t]) * state + b[:, t]
            ys.append(state)
        h = h + torch.stack(ys, 1)
        g = h @ p[f"{k}.gate"].t()
        h = h + (torch.nn.functional.silu(g) * (h @ p[f"{k}.up"].t())) @ p[f"{k}.down"].t()
    logits = h @ p["head"].t()
    return torch.nn.functional.cross_entropy(logits.flatten(0, 1), targets.flatten(), ignore_index=-100)


def test_runs():
    import train_recurrent_lm as example
    losses, held_out, out = example.main(steps=4, vocab=67, dim=64, layers=2, rows=2, length=100, verbose=False)
    assert losses.shape == (4,) and torch.isfinite(losses).all() and torch.isfinite(held_out)
    assert out.shape == (2, 8) and int(out.min()) >= 0 and int(out.max()) < 67


@pytest.mark.parametrize("rows,length", [(2, 70), (1, 5), (3, 33)])
def test_gradients_against_autograd(rows, length):
    import train_recurrent_lm as example
    vocab, dim, layers = 61, 32, 2
    params = example.init(vocab, dim, layers, hidden=48, seed=1)
    gen = torch.Generator(device="cuda").manual_seed(2)
    ids, targets, seq = example.documents(vocab, rows, length, gen)()
    if length >= 20:
        seq[:, length // 2:] += 1          # a document starts inside the row in any case
    loss, grads = example.Model(params, torch.float32).loss_and_grads(ids, targets, seq)
    ref = {k: v.double().cpu().requires_grad_() for k, v in params.items()}
    want = reference_loss(ref, ids.cpu(), targets.cpu(), seq.cpu(), layers)
    want.backward()
    assert abs(float(loss) - want.item()) <= 1e-5 * want.item()
    assert set(grads) == set(params)
    for k, g in grads.items():
        r = ref[k].grad
        assert g.shape == r.shape
        assert float((g.double().cpu() - r).norm()) <= 4e-4 * float(r.norm()), k


def test_bf16_gradients():
    """The same model in bfloat16, against float64 autograd of the rounded weights: a gradient is as far off as the
    roundings of the activations on its way make it, a few units of 2^-8 per layer: 0.06 (2-norm)."""
    import train_recurrent_lm as example
    params = example.init(64, 64, 2, seed=3)
    model = example.Model(params)
    ids, targets, seq = example.documents(64, 2, 90, torch.Generator(device="cuda").manual_seed(4))()
    loss, grads = model.loss_and_grads(ids, targets, seq)
    ref = {k: v.double().cpu().requires_grad_() for k, v in model.p.items()}
    want = reference_loss(ref, ids.cpu(), targets.cpu(), seq.cpu(), 2)
    want.backward()
    assert abs(float(loss) - want.item()) <= 0.02 * want.item()
    for k, g in grads.items():
        assert float((g.double().cpu() - ref[k].grad).norm()) <= 0.06 * float(ref[k].grad.norm()), k


def test_steps_continue_the_forward_pass():
    import train_recurrent_lm as example
    model = example.Model(example.init(61, 32, 2, hidden=48, seed=5), torch.float32)
    ids = torch.randint(0, 61, (3, 40), generator=torch.Generator().manual_seed(6)).cuda()
    whole = model.forward(ids)
    states = []
    model.forward(ids[:, :30].contiguous(), states=states)
    for t in range(30, 40):
        h = model.step(ids[:, t].contiguous(), states)
        assert float((h - whole[:, t]).norm() / whole[:, t].norm()) <= 4e-5


def test_no_call_of_the_example_drops_its_sequences(monkeypatch):
    """Training, the held-out loss and the prompt all work on packed rows: every call names their sequences."""
    import train_recurrent_lm as example
    calls = []

    def recurrence(v, *args, **kw):
        seq = kw.get("seq_idx")
        calls.append(seq is not None and tuple(seq.shape) == tuple(v.shape[:2]))
        return gated_recurrence(v, *args, **kw)

    monkeypatch.setattr(example, "gated_recurrence", recurrence)
    example.main(steps=2, vocab=67, dim=64, layers=2, rows=2, length=100, verbose=False)
    assert len(calls) == 2 * (2 + 1 + 1) and all(calls)


def test_packed_prompt_continues_its_last_document():
    """The states after a packed prompt, and what follows from them, are those of each row's last document alone.  (float32;
    the same steps in other tiles: each layer's states are within 4e-5, as in the test above.)"""
    import train_recurrent_lm as example
    model = example.Model(example.init(61, 32, 2, hidden=48, seed=7), torch.float32)
    ids = torch.randint(0, 61, (3, 50), generator=torch.Generator().manual_seed(8)).cuda()
    seq = torch.zeros((3, 50), dtype=torch.int32, device="cuda")
    last = (20, 0, 49)                    # where each row's last document starts
    seq[0, 7:], seq[0, 20:], seq[2, 49:] = 1, 2, 1
    packed_states = []
    h = model.forward(ids, seq, states=packed_states)
    follow = example.generate(model, ids, 6, seq)
    for row, start in enumerate(last):
        alone = ids[row:row + 1, start:].contiguous()
        states = []
        end = model.forward(alone, states=states)[0, -1]
        assert float((h[row, -1] - end).norm() / end.norm()) <= 4e-5
        for p, q in zip(packed_states, states):
            assert float((p[row] - q[0]).norm() / q[0].norm()) <= 4e-5
        assert torch.equal(follow[row], example.generate(model, alone, 6)[0])
