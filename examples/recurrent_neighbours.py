"""A recurrent next-token model that learns from its neighbours and answers with their drafts: the index, the recurrence,
the clipping of gradients and the verification of drafts together.

A token's row of one table enters the context, its row of another says how much of the context it keeps: the contexts
of a text are one `gated_scan` over it.  As in `neighbour_language_model.py` the neighbours of a context (`DCI.query`) are the
teacher of `distill_step`; the gradients go back through the recurrence (autograd) into both tables and are clipped by
their common norm (`clip_grads`).

To answer, the tokens that followed the nearest context in the corpus are a draft.  The model reads the draft in one call
of the recurrence, from the state that it keeps, and `verify_drafts` says which of its tokens stand and what follows; the state moves on by
as many tokens (`gated_scan` with lengths, in place).  What comes out is distributed as if the model had been asked
token by token.

    python examples/recurrent_neighbours.py
"""
import os
import sys

import torch

if __name__ == "__main__":
    sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
    sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
import dciknn_cuda_amd as D
from neighbour_language_model import corpus


class RecurrentModel:
    """table, gates and out [vocab, dim]; texts are read in windows from a state of zeros."""

    def __init__(self, vocab, dim, neighbours=16, seed=0, device="cuda"):
        g = torch.Generator(device=device).manual_seed(seed)
        self.table = torch.randn(vocab, dim, generator=g, device=device).requires_grad_()
        self.gates = (0.1 * torch.randn(vocab, dim, generator=g, device=device)).requires_grad_()
        self.out = (0.01 * torch.randn(vocab, dim, generator=g, device=device)).requires_grad_()
        self.velocity = [torch.zeros_like(w) for w in self.weights()]
        self.neighbours, self.dim = neighbours, dim
        self.dci = D.DCI(dim, num_comp_indices=2, num_simp_indices=7, bs=20, ts=10, seed=seed)

    def weights(self):
        return self.table, self.gates, self.out

    def contexts(self, tokens, state=None, lengths=None, last=None):
        """([batch, length, dim], the states behind): tokens [batch, length]."""
        return D.gated_scan(D.embed(self.table, tokens), D.embed(self.gates, tokens), state, lengths=lengths, last=last)

    @torch.no_grad()
    def index(self, windows):
        """All contexts of a corpus [windows, length + 1] but each window's last, and what follows them."""
        self.keys = self.contexts(windows[:, :-1])[0].reshape(-1, self.dim)        # borrowed by the index
        self.text, self.length = windows, windows.shape[1] - 1
        self.dci.clear()
        self.dci.add(self.keys)

    def teacher(self, contexts, sharpness):
        ids, dists = self.dci.query(contexts.detach(), self.neighbours, 200, return_int=True)
        at = ids.clamp(min=0).long()
        tokens = self.text[at // self.length, at % self.length + 1]
        return torch.where(ids >= 0, tokens, -1), -sharpness * dists * dists

    def gradients(self, windows, sharpness=4.0):
        """(mean loss, gradients by the weights) on windows [batch, length + 1]."""
        h = self.contexts(windows[:, :-1])[0].reshape(-1, self.dim)
        logits = h @ self.out.t()
        ids, teacher = self.teacher(h, sharpness)
        weights = torch.full((len(h),), 1.0 / len(h), device=h.device)
        losses, grad = D.distill_step(logits.detach(), ids, teacher, weights)
        return losses.mean(), torch.autograd.grad(logits, self.weights(), grad)

    def step(self, windows, rate, max_norm, momentum=0.9):
        """One step of gradient descent with momentum; (loss, norm of the gradients before they were clipped)."""
        loss, grads = self.gradients(windows)
        norm = D.clip_grads(grads, max_norm)
        with torch.no_grad():
            for weight, velocity, by_weight in zip(self.weights(), self.velocity, grads):
                weight -= rate * velocity.mul_(momentum).add_(by_weight)
        return loss, norm

    @torch.no_grad()
    def draft(self, state, k):
        """The k tokens that followed each state's nearest context in the corpus, -1 where its window ends: [batch, k]."""
        ids = self.dci.query(state, 1, 200, return_int=True)[0][:, :1].long()
        place = ids.clamp(min=0) % self.length + torch.arange(1, k + 1, device=state.device)
        tokens = self.text[(ids.clamp(min=0) // self.length), place.clamp(max=self.length)]
        return torch.where((ids >= 0) & (place <= self.length), tokens, -1)

    @torch.no_grad()
    def answer(self, prompts, count, drafts=4, temperature=1.0, seed=0):
        """(at least `count` tokens behind each of prompts [batch, length], how many calls of the model they took).

        The state is kept before the last token that is known, which is read with the drafts."""
        g = torch.Generator(device=prompts.device).manual_seed(seed)
        batch = len(prompts)
        state = self.contexts(prompts[:, :-1])[1] if prompts.shape[1] > 1 else torch.zeros(batch, self.dim, device=prompts.device)
        token, out, calls = prompts[:, -1:], [[] for _ in range(batch)], 0
        while min(len(o) for o in out) < count:
            here, _ = self.contexts(token, state)
            guess = self.draft(here[:, 0], drafts)
            read = torch.cat([token, guess], 1)
            h, _ = self.contexts(read, state)
            uniforms = torch.rand(batch, drafts + 1, generator=g, device=prompts.device)
            tokens, accepted, _ = D.verify_drafts(h @ self.out.t(), guess, uniforms, temperature=temperature)
            self.contexts(read, state, lengths=accepted + 1, last=state)
            token = tokens.gather(1, accepted[:, None].long()).long()
            calls += 1
            for row, kept, mine in zip(tokens.tolist(), accepted.tolist(), out):
                mine += row[:kept + 1]
        self.state, self.token = state, token
        return out, calls


def train(vocab=300, dim=64, length=64, windows=256, batch=32, steps=80, reindex=10, rate=3.0, max_norm=0.2, seed=0, say=print):
    """The model, and its mean log probability of held-out text before and after."""
    text = corpus(vocab, windows * (length + 1), seed + 2).view(windows, length + 1)
    held_out = corpus(vocab, 40 * (length + 1), seed + 3).view(40, length + 1)
    model = RecurrentModel(vocab, dim, seed=seed)

    @torch.no_grad()
    def score():
        logits = model.contexts(held_out[:, :-1])[0] @ model.out.t()
        return D.token_logprobs(logits, held_out[:, 1:])[0].mean().item()

    before = score()
    g = torch.Generator(device="cuda").manual_seed(seed)
    for i in range(steps):
        if i % reindex == 0:
            model.index(text)
        loss, norm = model.step(text[torch.randint(0, windows, (batch,), generator=g, device="cuda")], rate, max_norm)
        if i % 20 == 19:
            say("step %d: loss %.3f, norm of the gradients %.3f" % (i + 1, loss.item(), norm.item()))
    model.index(text)
    after = score()
    say("log probability of held-out text: %.3f before, %.3f after" % (before, after))
    out, calls = model.answer(held_out[:8, :20], 40)
    say("%d tokens or more behind 8 prompts by %d calls of the model" % (min(len(o) for o in out), calls))
    return model, before, after


if __name__ == "__main__":
    train()
