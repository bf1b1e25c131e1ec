"""The example that uses the index and the token operators together."""
import os
import sys

import pytest
import torch

pytestmark = pytest.mark.gpu
sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples"))


def test_neighbours_teach_the_model(gpu):
    import neighbour_language_model as N
    before, after = N.train(say=lambda line: None)
    # a chance token is among four of 500 in 0.8 % of the cases; a successor follows in 95 % of them
    assert after[0] > before[0] + 1.0 and after[2] > 0.5


def test_a_step_is_what_torch_computes(gpu):
    """Table and output layer after one step, against torch's own lookup, softmax and autograd in 64 bits."""
    import neighbour_language_model as N
    text = N.corpus(50, 400, 5)
    model = N.NeighbourModel(50, 16, seed=3)
    model.index(text)
    ends = torch.arange(0, 399, 7, device="cuda")
    table, out = (w.detach().double().requires_grad_() for w in (model.table, model.out))
    at = ends[:, None] + torch.arange(1 - model.span, 1, device="cuda")
    rows = table[text[at.clamp(min=0)]] * (at >= 0)[:, :, None] * 16 ** -0.5
    h = (rows * model.decay.double()[:, None]).sum(1)
    ids, teacher = model.teacher(h.float(), 4.0)
    q = torch.softmax(teacher.double(), 1)
    logp = torch.log_softmax(h @ out.t(), 1)
    loss = (q * (torch.log(q.clamp(min=1e-300)) - logp.gather(1, ids.clamp(min=0)))).sum(1).mean()
    loss.backward()
    got = model.step(text, ends, rate=2.0)
    assert abs(got.item() - loss.item()) < 1e-3
    # products of 16 to 50 terms and sums over 57 rows in 32 bits: some 1e-5 of the largest; ten times that
    for weight, expected in ((model.table, table), (model.out, out)):
        want = expected.detach() - 2.0 * expected.grad
        assert (weight.detach().double() - want).abs().max() < 2.0 * 1e-4 * expected.grad.abs().max() + 1e-6
