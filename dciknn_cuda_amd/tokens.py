"""Operators of programs that train or serve a model on the rows and neighbours that `DCI` indexes
and finds: rows taken by ids and the gradient by their table, log probabilities of tokens, and
the loss against a teacher that is known by its best tokens, as a query's neighbours are.

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
