"""A small next-token model taught by its own nearest neighbours: the index and the operators on tokens together.

A context is the decayed sum of its last tokens' rows of an embedding table (`embed`), its logits are their products
with the rows of an output layer.  All contexts of a corpus are indexed (`DCI.add`); the neighbours of a batch's contexts
(`DCI.query`) name the tokens that followed there, their distances are the logits of a teacher, and the model
learns that distribution (`distill_step`).  The gradient goes on through the lookup into the table (`embed`'s
backward is `embed_grad`), and the index follows the table every few steps.  Held-out text is scored with
`token_logprobs`.

    python examples/neighbour_language_model.py
"""
import os
import sys

import torch

if __name__ == "__main__":
    sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
import dciknn_cuda_amd as D


def corpus(vocab, length, seed):
    """Tokens of a chain in which every token has four likely successors."""
    g = torch.Generator().manual_seed(seed)
    follows = torch.randint(0, vocab, (vocab, 4), generator=torch.Generator().manual_seed(1))
    picks = torch.randint(0, 4, (length,), generator=g)
    stray = torch.rand(length, generator=g) < 0.05
    random = torch.randint(0, vocab, (length,), generator=g)
    out = torch.zeros(length, dtype=torch.int64)
    for i in range(1, length):
        out[i] = random[i] if stray[i] else follows[out[i - 1], picks[i]]
    return out.cuda()


class NeighbourModel:
    """table and out [vocab, dim]; a context is the last `span` tokens."""

    def __init__(self, vocab, dim, span=2, neighbours=16, seed=0, device="cuda"):
        g = torch.Generator(device=device).manual_seed(seed)
        self.table = torch.randn(vocab, dim, generator=g, device=device).requires_grad_()
        self.out = (0.01 * torch.randn(vocab, dim, generator=g, device=device)).requires_grad_()
        self.velocity = [torch.zeros_like(self.table), torch.zeros_like(self.out)]
        self.decay = 0.5 ** torch.arange(span - 1, -1, -1, device=device)       # the last token counts most
        self.span, self.neighbours = span, neighbours
        self.dci = D.DCI(dim, num_comp_indices=2, num_simp_indices=7, bs=20, ts=10, seed=seed)

    def contexts(self, tokens, ends):
        """[n, dim] for the positions `ends` of their last tokens; places before the text are empty slots."""
        at = ends[:, None] + torch.arange(1 - self.span, 1, device=ends.device)
        ids = torch.where(at >= 0, tokens[at.clamp(min=0)], -1)
        rows = D.embed(self.table, ids, self.table.shape[1] ** -0.5)
        return (rows * self.decay[:, None]).sum(1)

    def index(self, tokens):
        with torch.no_grad():
            ends = torch.arange(tokens.shape[0] - 1, device=tokens.device)
            self.keys = self.contexts(tokens, ends).contiguous()        # borrowed by the index
            self.next_tokens = tokens[1:]
        self.dci.clear()
        self.dci.add(self.keys)

    def teacher(self, contexts, sharpness):
        """Token ids and logits of the neighbours; empty slots stay so (id -1, logit -inf)."""
        ids, dists = self.dci.query(contexts.detach().contiguous(), self.neighbours, 200, return_int=True)
        tokens = torch.where(ids >= 0, self.next_tokens[ids.clamp(min=0).long()], -1)
        return tokens, -sharpness * dists * dists

    def step(self, tokens, ends, rate, sharpness=4.0, momentum=0.9):
        """One step of gradient descent with momentum; the mean loss."""
        h = self.contexts(tokens, ends)
        logits = h @ self.out.t()
        ids, teacher = self.teacher(h, sharpness)
        weights = torch.full(ends.shape, 1.0 / ends.shape[0], device=ends.device)
        losses, grad = D.distill_step(logits.detach(), ids, teacher, weights)
        grads = torch.autograd.grad(logits, (self.table, self.out), grad)
        with torch.no_grad():
            for weight, velocity, by_weight in zip((self.table, self.out), self.velocity, grads):
                weight -= rate * velocity.mul_(momentum).add_(by_weight)
        return losses.mean()

    @torch.no_grad()
    def score(self, tokens, top=4):
        """(mean log probability of the text, mean entropy, share of tokens among the `top` best)."""
        ends = torch.arange(tokens.shape[0] - 1, device=tokens.device)
        logits = self.contexts(tokens, ends) @ self.out.t()
        logp, entropy, best, _ = D.token_logprobs(logits, tokens[1:], top=top)
        return logp.mean().item(), entropy.mean().item(), (best == tokens[1:, None]).any(1).float().mean().item()


def train(vocab=500, dim=64, length=20_000, batch=2048, steps=60, reindex=10, rate=50.0, seed=0, say=print):
    """The scores of held-out text before and after."""
    text, held_out = corpus(vocab, length, seed + 2), corpus(vocab, 2000, seed + 3)
    model = NeighbourModel(vocab, dim, seed=seed)
    before = model.score(held_out)
    say("before: log probability %.3f, entropy %.3f, among the four best %.3f" % before)
    g = torch.Generator(device="cuda").manual_seed(seed)
    for i in range(steps):
        if i % reindex == 0:
            model.index(text)
        loss = model.step(text, torch.randint(0, length - 1, (batch,), generator=g, device="cuda"), rate)
        if i % 20 == 19:
            say("step %d: loss %.3f" % (i + 1, loss.item()))
    after = model.score(held_out)
    say("after:  log probability %.3f, entropy %.3f, among the four best %.3f" % after)
    return before, after


if __name__ == "__main__":
    train()
