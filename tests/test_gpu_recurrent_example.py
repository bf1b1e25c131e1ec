"""The recurrence, the clipping and the verification as a model uses them together, with the index."""
import os
import sys

import pytest
import torch

pytestmark = pytest.mark.gpu
sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples"))


def small(seed=3, vocab=40, dim=16, length=12, windows=30):
    import recurrent_neighbours as R
    model = R.RecurrentModel(vocab, dim, seed=seed)
    text = R.corpus(vocab, windows * (length + 1), seed).view(windows, length + 1)
    model.index(text)
    return model, text


def test_it_runs(gpu):
    import recurrent_neighbours as R
    lines = []
    model, before, after = R.train(vocab=50, dim=16, length=16, windows=40, batch=8, steps=20, say=lines.append)
    assert len(lines) == 3 and all(torch.isfinite(w).all() for w in model.weights()) and before == before and after == after


def test_gradients_are_what_torch_computes(gpu):
    """Of one step, by torch's own lookup, a loop over the tokens, softmax and autograd in 64 bits."""
    model, text = small()
    windows = text[:6]
    weights = [w.detach().double().requires_grad_() for w in model.weights()]
    table, gates, out = weights
    x, a = table[windows[:, :-1]], torch.sigmoid(gates[windows[:, :-1]])
    h, rows = torch.zeros(6, 16, device="cuda", dtype=torch.float64), []
    for t in range(x.shape[1]):
        h = a[:, t] * h + (1 - a[:, t]) * x[:, t]
        rows.append(h)
    h = torch.stack(rows, 1).reshape(-1, 16)
    ids, teacher = model.teacher(h.float(), 4.0)
    q = torch.softmax(teacher.double(), 1)
    logp = torch.log_softmax(h @ out.t(), 1)
    loss = (q * (torch.log(q.clamp(min=1e-300)) - logp.gather(1, ids.clamp(min=0)))).sum(1).mean()
    want = torch.autograd.grad(loss, weights)
    got_loss, got = model.gradients(windows)
    assert abs(got_loss.item() - loss.item()) < 1e-3
    # products of 16 to 50 terms and sums over some tokens in 32 bits: some 1e-5 of the largest; ten times that
    for mine, right in zip(got, want):
        assert (mine.double() - right).abs().max() < 1e-4 * right.abs().max()
    norm = torch.cat([w.flatten() for w in want]).norm()
    before, velocity = [w.detach().clone() for w in model.weights()], 0.5 * norm.item()
    _, got_norm = model.step(windows, 2.0, velocity)
    assert abs(got_norm.item() - norm.item()) < 1e-4 * norm.item()
    for w, b, right in zip(model.weights(), before, want):
        moved = -2.0 * 0.5 * right                       # a first step: half the gradient, times the rate
        assert (w.detach().double() - b.double() - moved).abs().max() < 3e-4 * right.abs().max() + 1e-6


def test_state_follows_what_was_accepted(gpu):
    """After any number of calls the state is that of the prompt and the answer read from the start."""
    model, text = small()
    prompts = text[:5, :7]
    out, calls = model.answer(prompts, 15, drafts=3, temperature=0.5, seed=1)
    assert calls <= 15 and all(len(o) >= 15 and all(0 <= t < 40 for t in o) for o in out)
    for b in range(5):
        said = torch.tensor(prompts[b].tolist() + out[b], device="cuda")
        assert said[-1] == model.token[b, 0]
        _, want = model.contexts(said[None, :-1])
        # up to 60 tokens of 16 half steps of values up to 5, twice
        assert (model.state[b] - want[0]).abs().max() < 2 * 60 * 16 * 5 * 2.0 ** -24


def test_drafts_change_nothing_but_the_number_of_calls(gpu):
    """At a temperature at which the model is certain, token by token and by drafts are the same."""
    model, text = small()
    with torch.no_grad():
        model.out.mul_(100.0)
    one, calls_one = model.answer(text[:6, :5], 12, drafts=0, temperature=1e-3)
    many, calls_many = model.answer(text[:6, :5], 12, drafts=4, temperature=1e-3)
    assert calls_one == 12 and calls_many <= calls_one
    for a, b in zip(one, many):
        assert a[:12] == b[:12]


def test_answers_are_distributed_as_the_model_says(gpu):
    """The first token behind 20000 equal prompts, with drafts from the index."""
    model, text = small()
    with torch.no_grad():
        model.out.mul_(20.0)
    n = 20_000
    prompts = text[:1, :6].expand(n, 6).contiguous()
    out, _ = model.answer(prompts, 1, drafts=2, seed=4)
    first = torch.tensor([o[0] for o in out])
    with torch.no_grad():
        h, _ = model.contexts(prompts[:1])
        p = torch.softmax((h[:, -1] @ model.out.t()).double(), 1)[0].cpu()
    got = torch.bincount(first, minlength=40).double() / n
    # six standard deviations of each share
    assert ((got - p).abs() < 6 * (p * (1 - p) / n).sqrt() + 1e-9).all()
