"""Operators of programs that train or serve a model on the rows and neighbours that `DCI` indexes
and finds: rows taken by ids and the gradient by their table, contexts of texts by a recurrence, log probabilities of tokens,
the loss against a teacher that is known by its best tokens, as a query's neighbours are, gradients clipped by their
norm, and drafted tokens, as neighbours propose them, verified against the model.

The tensors are float32, float16 or bfloat16 cuda tensors; sums are formed in 32 bits and results
rounded once.  Rows may start anywhere and be at any one distance from each other, their own elements are
contiguous.  (`logits[:, :-1]` of a batch is at two distances and refused: give all rows, with targets
or teacher's ids of -1 in the last ones, whose log probabilities, losses and gradients by them are 0;
entropies are of all rows.)  Ids are int32 or int64 (`DCI.query(..., return_int=True)` returns int32), ids and
factors of any strides.  An id below 0 marks an empty slot, as `DCI.query` leaves them; an id beyond the
table or the vocabulary is never accessed and gives NaN.  Work goes to torch's current stream, without a
wait; gradients are taken through torch.autograd, once, and backward: a tangent of forward mode is
refused.  Wrong types raise TypeError, wrong shapes and values ValueError.  The reference, a search engine
alone, has no counterpart.
"""
from . import _dci_cuda as _ext   # built by `python -m dciknn_cuda_amd.build`; no fallback


def embed(table, ids, scale=1.0):
    """`scale * table[ids]`: table [rows, dim], ids of any shape -> [*ids.shape, dim].

    An empty slot gives a row of zeros, an id beyond the table one of NaN.  Differentiable by
    `table` (see `embed_grad`)."""
    return _ext._embed(table, ids, scale)


def embed_grad(grad, ids, num_rows, scale=1.0, *, out=None):
    """The gradient of `embed` by its table: [num_rows, dim], row r the sum of `scale * grad[i]`
    over the i with ids[i] = r; empty slots and ids beyond the table add nothing.

    The sum's order depends on the ids alone: the same input gives the same bits.  With `out`
    ([num_rows, dim], contiguous, of grad's type or float32) the sums are added to it and it is returned; its
    rows without ids are not touched.  No gradient is formed by `grad`: one that requires it is refused."""
    return _ext._embed_grad(grad, ids, num_rows, scale, out)


def token_logprobs(logits, targets, top=0, temperature=1.0):
    """(logprobs, entropy) of the rows of logits [..., vocab] for targets [...], both float32, with
    p = softmax(logits / temperature): log p[target] and -sum p log p.

    With top > 0 (up to 64) also (top_ids, top_logprobs) [..., top]: the largest logits in descending order, equal
    ones by index, those of -inf or NaN last.  A target below 0 gives 0; a row of nothing but
    -inf has log probabilities of -inf and entropy 0.  Differentiable by `logits` through logprobs and
    entropy; a row whose two factors are 0 has gradient 0 whatever it holds."""
    return _ext._token_logprobs(logits, targets, top, temperature)


def distill_loss(logits, ids, teacher, temperature=1.0):
    """Losses [...] (float32) of the rows of logits [..., vocab] against a teacher's best tokens:
    ids and teacher [..., slots], its logits; up to 1024 slots.

    With q = softmax(teacher / temperature) over a row's filled slots (id not below 0, logit above -inf) and
    p = softmax(logits / temperature): sum_j q_j (log q_j - log p[ids_j]).  An id may stand in several
    slots; without filled slots the loss is 0.  Neighbours are a teacher by
    `ids, dists = dci.query(..., return_int=True)` and `teacher = -dists`.  Differentiable by `logits`."""
    return _ext._distill_loss(logits, ids, teacher, temperature)


def distill_step(logits, ids, teacher, weights=None, temperature=1.0, *, out=None):
    """(losses, grad): `distill_loss` and the gradient of `(weights * losses).sum()` by logits in
    one call, which reads the logits once where rows fit the chip; no autograd graph.

    weights [...] float32, ones if not given; a row with weight 0 has gradient 0 whatever it
    holds.  `out`: where the gradient goes, also `logits` itself; a leaf that requires a gradient, or anything
    else that does, is refused."""
    return _ext._distill_step(logits, ids, teacher, weights, temperature, out)


def gated_scan(x, gates, state=None, *, decay=False, lengths=None, offsets=None, last=None):
    """(h, last) of a linear recurrence over the tokens of sequences, each channel by itself: with a = sigmoid(gates)
    h_t = a_t * h_(t-1) + (1 - a_t) * x_t, with `decay` a = gates and h_t = a_t * h_(t-1) + x_t.

    x [batch, length, dim], with `lengths` [batch] the tokens of each (h is 0 behind them, and nothing there is looked
    at), or x [tokens, dim], one sequence or, with `offsets` [sequences + 1], those between them one behind the other.  gates are of
    x's shape, or [dim] for all tokens; state [sequences, dim] float32 is what stands before the first tokens, zeros if not given.  h is of x's
    shape and type, last [sequences, dim] float32 the state behind the last tokens.  The channels of a token are next to one another, tokens and
    rows at any distances.  A server's step is a length of 1, with `last=state` in place.  States are in 32 bits; one that is not finite
    leaves none finite behind it in its sequence.  Decays may be of any size; stretches of a hundred tokens that may grow 2**100 times are slow.  Differentiable by x, gates and state, not with `last`."""
    return _ext._gated_scan(x, gates, state, decay, lengths, offsets, last)


def grad_norm(grads, scale=1.0):
    """The norm of a model's gradients times `scale`, all of them as one vector: a float32 tensor of no dimensions.

    grads: tensors of any of the types and shapes, mixed, each dense (in any order of its dimensions).  Squares are summed in 64 bits in an
    order that depends on the shapes alone.  Of no gradients it is 0, on the CPU."""
    return _ext._grad_norm(list(grads), scale)


def clip_grads(grads, max_norm, scale=1.0, *, out=None):
    """Multiplies the gradients, in their place or into `out`, by `scale * min(1, max_norm / norm)`; returns the norm before
    clipping, `grad_norm(grads, scale)`, without waiting for it.

    `scale` undoes a loss's factor.  out: for each gradient a tensor of its shape and strides, of its type or float32; no two
    tensors of a call may share memory.  A norm that is infinite or NaN clips nothing (out = grads * scale)."""
    return _ext._clip_grads(list(grads), max_norm, scale, None if out is None else list(out))


def verify_drafts(logits, drafts, uniforms, ids=None, teacher=None, temperature=1.0):
    """(tokens, accepted, logprobs): which drafted tokens stand before the model's probabilities, and the token behind them.

    drafts [batch, k] (0 to 256, the first below 0 ends a sequence's), logits [batch, k + 1, vocab] with row i what the model says
    behind i of them: p = softmax(logits / temperature).  ids and teacher [batch, k, slots]: the tokens a draft was drawn from and their
    logits, q = softmax(teacher) over the filled slots, as in `distill_loss` (for tokens drawn from a model's best, what `token_logprobs`
    returns for them); without them a draft was named for certain, as by the nearest neighbour.  uniforms [batch, k + 1] float32 in [0, 1):
    draft i stands while uniforms[i] * q(draft) < p(draft); the next token is drawn by uniforms[k] from max(p - q, 0) of the first that does not,
    else from the last p, as the first at which the running sum of the weights is above that share of all.
    The tokens are distributed as if drawn from the model one by one.

    tokens [batch, k + 1] int32: the accepted [batch] drafts, the next token, -1 behind it; logprobs float32: their log p,
    0 behind them.  A row without probabilities (NaN, +inf, nothing but -inf) gives -1 with NaN.  Decided in 64 bits, at the temperature
    rounded to 32 as everywhere here; what is left of a token within 1e-13 of what q takes off is nothing, and where nothing is left p is
    drawn from."""
    return _ext._verify_drafts(logits, drafts, uniforms, ids, teacher, temperature)
