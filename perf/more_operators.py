"""What the time of the recurrence, the clipping of gradients and the verification of drafts is measured on.

A case is one call, or a call and its gradient, that a program makes which trains a recurrent next-token model on
rows and neighbours that `DCI` indexes and finds, or serves it with drafts that the neighbours propose:

  scan        a gated linear recurrence over the tokens of sequences (`gated_scan`)
  scantrain   the same and its gradients by inputs, gates and first states
  norm        the norm of all gradients of a model (`grad_norm`)
  clip        gradients clipped by that norm, into others or in their place (`clip_grads`)
  verify      drafted tokens kept or replaced by the model's probabilities (`verify_drafts`)

With `own` false they are computed in their plain form by elementary torch operations, in 32 bits; sums over all
gradients, and probabilities that decide on a token, in 64.
"""
import math
import random

import torch

own = False

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
BYTES = {"f32": 4, "bf16": 2, "f16": 2}


def _scan(name, op, batch, length, dim, dtype="bf16", decay=False, shared=False, form="batch", state=True):
    """`form` batch: [batch, length, dim]; lengths: of these a number of tokens each; packed: `length` tokens in all
    of `batch` sequences one behind the other, [length, dim].  shared: one gate for all tokens of a channel."""
    c = dict(op=op, batch=batch, length=length, dim=dim, dtype=dtype, decay=decay, shared=shared, form=form, state=state)
    if name:
        c["name"] = name
    return c


def _grads(name, op, tensors, largest, dim, dtype="bf16", into="same", scale=1.0):
    """`tensors` gradients: matrices of up to `largest` rows by `dim`, among them rows of `dim`, with `dim` 0 vectors of
    any length up to `largest`.  into: same or f32 (other tensors, of which type), place (in place, norm within bounds);
    what is written are parts of one buffer, as optimizers and data-parallel training keep them."""
    c = dict(op=op, tensors=tensors, largest=largest, dim=dim, dtype=dtype, into=into, scale=scale)
    if name:
        c["name"] = name
    return c


def _verify(name, batch, drafts, vocab, slots=0, dtype="bf16", temperature=1.0, ids64=True):
    """slots: of the distribution a draft was drawn from, 0: it was named for certain."""
    c = dict(op="verify", batch=batch, drafts=drafts, vocab=vocab, slots=slots, dtype=dtype, temperature=temperature, ids64=ids64)
    if name:
        c["name"] = name
    return c


def listed():
    return [
        # One step of a server: the tokens of 32 sequences.
        _scan("scan-step", "scan", 32, 1, 4096),
        # Long prompts of a server's batch, one behind the other.
        _scan("scan-prompt", "scan", 6, 65_536, 4096, form="packed"),
        # The contexts of the example's corpus: 20 000 tokens, rows of 64, a decay for each channel, and its gradient.
        _scan("scan-corpus", "scantrain", 1, 20_000, 64, dtype="f32", decay=True, shared=True, state=False),
        # A training step.
        _scan("scan-train", "scantrain", 8, 4096, 2048, state=False),
        # Documents of any length with rows of odd length, one behind the other.
        _scan("scan-ragged", "scantrain", 45, 30_011, 1023, dtype="f16", form="packed"),
        # The example's table and output layer.
        _grads("clip-small", "clip", 2, 500, 64, dtype="f32"),
        # Gradients in 16 bits of a model of some 200 million weights, clipped into those of 32 bits that an optimizer takes.
        _grads("clip-model", "clip", 120, 8192, 2048, into="f32"),
        # A step whose gradients are within the bound, in their place.
        _grads("clip-within", "clip", 300, 4096, 1024, dtype="f32", into="place"),
        # Many gradients of all sizes under a loss that was scaled up.
        _grads("norm-ragged", "norm", 1000, 1_000_000, 0, dtype="f16", scale=1.0 / 1024),
        # A server's step: four sequences with four drafts, the next tokens of the nearest neighbour.
        _verify("verify-step", 4, 4, 131_072),
        # A batch with drafts drawn from ten neighbours' next tokens, a vocabulary of odd length.
        _verify("verify-ragged", 17, 3, 50_001, slots=10, dtype="f16", temperature=0.7, ids64=False),
        # A large batch with drafts drawn from 64 best tokens.
        _verify("verify-batch", 64, 7, 131_072, slots=64),
    ]


def _spread(rng, lo, hi):
    """A whole number in [lo, hi], even over its logarithm."""
    return min(hi, max(lo, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    op = rng.choice(["scan", "scan", "scantrain", "scantrain", "scantrain", "norm", "clip", "clip", "verify", "verify", "verify"])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    if op in ("scan", "scantrain"):
        dim = _spread(rng, 16, 8192)
        if rng.random() < 0.7:                     # most rows are whole 16-byte words
            dim = (dim + 7) // 8 * 8
        form = rng.choice(["batch", "batch", "lengths", "packed"])
        most = (1 << 27 if op == "scan" else 1 << 26) // dim * 2 // BYTES[dtype]
        length = min(most, _spread(rng, 1, 65_536))
        batch = _spread(rng, 1, 256)
        if form != "packed":
            batch = max(1, min(batch, most // length))
        else:
            batch = min(batch, max(1, length // 4))
        return _scan(None, op, batch, length, dim, dtype, rng.random() < 0.4, rng.random() < 0.25, form, rng.random() < 0.5)
    if op in ("norm", "clip"):
        dim = rng.choice([0, _spread(rng, 16, 4096)])
        largest = _spread(rng, 100, 10_000) if dim else _spread(rng, 100, 1_000_000)
        tensors = min(_spread(rng, 1, 2000), max(1, (1 << 28) // (largest * max(dim, 1))))
        return _grads(None, op, tensors, largest, dim, dtype, rng.choice(["same", "f32", "place"]), rng.choice([1.0, 1.0, 2.0 ** -10]))
    vocab = _spread(rng, 1000, 262_144)
    if rng.random() < 0.6:                         # most vocabularies are padded to whole lines
        vocab = (vocab + 63) // 64 * 64
    drafts = rng.choice([0, 1, 2, 3, 4, 5, 7, 10, 16])
    batch = max(1, min(_spread(rng, 1, 256), (1 << 26) // (vocab * (drafts + 1)) * 2 // BYTES[dtype]))
    slots = rng.choice([0, _spread(rng, 2, 128)]) if drafts else 0
    return _verify(None, batch, drafts, vocab, slots, dtype, rng.choice([1.0, 1.0, 0.7, 1.5]), rng.random() < 0.6)


def _shapes(case):
    """Of the gradients: from the case alone."""
    rng = random.Random(case["tensors"] * 7 + case["largest"])
    shapes = []
    for i in range(case["tensors"]):
        if not case["dim"]:
            shapes.append((_spread(rng, 1, case["largest"]),))
        elif i % 3 == 2:
            shapes.append((case["dim"],))
        else:
            shapes.append((max(1, case["largest"] >> rng.choice([0, 1, 2, 3])), case["dim"]))
    if not case["dim"] or case["tensors"] < 3:
        shapes[0] = (case["largest"], case["dim"]) if case["dim"] else (case["largest"],)
    return shapes


def _cuts(case, gen):
    """Offsets of packed sequences: any lengths, some of them none."""
    n, tokens = case["batch"], case["length"]
    inner = (torch.rand(n - 1, generator=gen, device="cuda", dtype=torch.float64) * tokens).long().sort().values
    ends = torch.tensor([0, tokens], device="cuda")
    return torch.cat([ends[:1], inner, ends[1:]]).int()


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    dtype = TYPES[case["dtype"]]
    s = dict(case=case)

    def randn(*shape):
        return torch.randn(*shape, generator=gen, device="cuda")

    def rand(*shape):
        return torch.rand(*shape, generator=gen, device="cuda")

    if case["op"] in ("scan", "scantrain"):
        n, t, d = case["batch"], case["length"], case["dim"]
        shape = (t, d) if case["form"] == "packed" else (n, t, d)
        s["x"] = torch.empty(shape, device="cuda", dtype=dtype).normal_(0.0, 1.0, generator=gen)
        gates = (d,) if case["shared"] else shape
        # a channel forgets within one to some hundred tokens
        if case["decay"]:
            s["gates"] = (1.0 - 0.5 ** (1.0 + 7.0 * rand(*gates))).to(dtype)
        else:
            s["gates"] = torch.empty(gates, device="cuda", dtype=dtype).normal_(2.0, 2.0, generator=gen)
        s["state"] = randn(n, d) if case["state"] else None
        s["lengths"] = s["offsets"] = None
        if case["form"] == "lengths":
            s["lengths"] = (rand(n) * (t + 1)).int()
        if case["form"] == "packed":
            s["offsets"] = _cuts(case, gen)
        if case["op"] == "scantrain":
            # (the sum over all tokens of a shared gate's has to fit 16 bits)
            share = 8.0 * (s["x"].numel() // d) ** -0.5 if case["shared"] else 1.0
            s["dh"], s["dlast"] = (randn(*shape) * share).to(dtype), randn(n, d) * share
            s["leaves"] = [s["x"], s["gates"]] + ([s["state"]] if case["state"] else [])
            for leaf in s["leaves"]:
                leaf.requires_grad_()
        return s
    if case["op"] in ("norm", "clip"):
        shapes = _shapes(case)
        s["grads"] = [(randn(*shape) * (0.01 / case["scale"] ** 0.5)).to(dtype) for shape in shapes]
        total = sum(math.prod(shape) for shape in shapes)
        # about a tenth of the norm, or above it
        s["max_norm"] = 0.01 * case["scale"] ** 0.5 * total ** 0.5 * (10.0 if case["into"] == "place" else 0.1)
        if case["into"] == "place":
            s["case"] = case = dict(case, scale=1.0)
            s["max_norm"] *= 1024.0
        if case["op"] == "clip":
            s["flat"] = torch.empty(total, device="cuda", dtype=torch.float32 if case["into"] == "f32" else dtype)
            parts = [part.view(shape) for part, shape in zip(s["flat"].split([math.prod(shape) for shape in shapes]), shapes)]
            if case["into"] == "place":
                s["grads"], s["out"] = [part.copy_(g) for part, g in zip(parts, s["grads"])], None
            else:
                s["out"] = parts
        return s
    n, k, v, slots = case["batch"], case["drafts"], case["vocab"], case["slots"]
    ids = torch.int64 if case["ids64"] else torch.int32
    z = torch.empty(n, k + 1, v, device="cuda").normal_(0.0, 2.5, generator=gen)
    right = (float(v) ** rand(n, k + 1, 1).double() - 1.0).long().clamp_(0, v - 1)
    z.scatter_add_(2, right, 6.0 + 8.0 * rand(n, k + 1, 1))
    s["logits"] = z.to(dtype)
    s["uniforms"] = rand(n, k + 1)
    s["ids"] = s["teacher"] = None
    drafts = torch.where(rand(n, k) < 0.8, right[:, :k, 0], (v * rand(n, k)).long())
    if slots:
        # neighbours' next tokens, the right one among them and some of them the same
        at = (float(v) ** rand(n, k, slots).double() - 1.0).long().clamp_(0, v - 1)
        at[:, :, 0] = right[:, :k, 0]
        s["teacher"] = -torch.sort(6.0 * rand(n, k, slots), dim=2).values
        chosen = (s["teacher"] - torch.log(-torch.log(rand(n, k, slots)))).argmax(2, keepdim=True)
        drafts = at.gather(2, chosen)[:, :, 0]
        s["ids"] = at.to(ids)
    # some sequences have fewer drafts
    fewer = (rand(n, 1) * 2 * (k + 1)).int()
    s["drafts"] = torch.where(torch.arange(k, device="cuda")[None, :] < fewer, drafts, -1).to(ids)
    return s


def _starts(s, tokens):
    """(sequence of each token, whether it is the first) of packed sequences."""
    t = torch.arange(tokens, device="cuda")
    of = torch.searchsorted(s["offsets"].long(), t, right=True) - 1
    return of, s["offsets"].long()[of] == t


def _doubling(a, b, dim):
    """h_t = a_t h_(t-1) + b_t along `dim`, by log2 of the length steps."""
    step, t = 1, a.shape[dim]
    while step < t:
        b = torch.cat([b.narrow(dim, 0, step), torch.addcmul(b.narrow(dim, step, t - step), a.narrow(dim, step, t - step), b.narrow(dim, 0, t - step))], dim)
        if 2 * step < t:
            a = torch.cat([a.narrow(dim, 0, step), a.narrow(dim, step, t - step) * a.narrow(dim, 0, t - step)], dim)
        step *= 2
    return b


def _plain_scan(s):
    case = s["case"]
    n, t, d, decay, dtype = case["batch"], case["length"], case["dim"], case["decay"], TYPES[case["dtype"]]
    packed = case["form"] == "packed"
    x, g = s["x"].detach().float(), s["gates"].detach().float()
    state = s["state"].detach() if case["state"] else torch.zeros(n, d, device="cuda")
    axis = 0 if packed else 1
    a = (g if decay else 1.0 / (1.0 + torch.exp(-g))).expand(x.shape)
    b = x if decay else x - a * x
    inside = None
    if packed:
        of, first = _starts(s, t)
        carry = torch.where(first[:, None], 0.0, a)
        start = torch.where(first[:, None], state[of], 0.0)
        lengths = (s["offsets"][1:] - s["offsets"][:-1]).long()
        ends = s["offsets"][1:].long() - 1
    else:
        first = torch.zeros(t, 1, dtype=torch.bool, device="cuda")
        first[0] = True
        carry, start = torch.where(first, 0.0, a), torch.where(first, state[:, None], 0.0)
        lengths = s["lengths"].long() if s["lengths"] is not None else torch.full((n,), t, device="cuda")
        ends = torch.arange(n, device="cuda") * t + lengths - 1
        if s["lengths"] is not None:
            inside = (torch.arange(t, device="cuda")[None, :] < lengths[:, None])[:, :, None]
    h = _doubling(carry, b + a * start, axis)
    if inside is not None:
        h = torch.where(inside, h, 0.0)
    some = (lengths > 0)[:, None]
    ends = ends.clamp(min=0)
    last = torch.where(some, h.reshape(-1, d)[ends], state)
    if case["op"] == "scan":
        return h.to(dtype), last
    # l_t = dh_t + a_(t+1) l_(t+1) within a sequence
    l = s["dh"].float()
    if inside is not None:
        l = torch.where(inside, l, 0.0)
    l = l.reshape(-1, d).index_add(0, ends, torch.where(some, s["dlast"], 0.0)).reshape(x.shape)
    back = torch.cat([carry.narrow(axis, 1, t - 1), torch.zeros_like(carry.narrow(axis, 0, 1))], axis)
    l = _doubling(back.flip(axis), l.flip(axis), axis).flip(axis)
    before = torch.where(first[:, None] if packed else first, start, torch.cat([torch.zeros_like(h.narrow(axis, 0, 1)), h.narrow(axis, 0, t - 1)], axis))
    dx, dg = (l, l * before) if decay else (l - a * l, l * (before - x) * a * (1.0 - a))
    if inside is not None:
        dg = torch.where(inside, dg, 0.0)
    if case["shared"]:
        dg = dg.reshape(-1, d).sum(0)
    out = [h.to(dtype), last, dx.to(dtype), dg.to(dtype)]
    if case["state"]:
        heads = (s["offsets"][:-1].long() if packed else torch.arange(n, device="cuda") * t).clamp(max=x.numel() // d - 1)
        out.append(torch.where(some, (a * l).reshape(-1, d)[heads], s["dlast"]))
    return tuple(out)


def _softmax(z):
    e = torch.exp(z - z.max(dim=-1, keepdim=True).values)
    return e / e.sum(dim=-1, keepdim=True)


def _plain_verify(s):
    case = s["case"]
    n, k, v = case["batch"], case["drafts"], case["vocab"]
    z = s["logits"].double() / case["temperature"]
    p = _softmax(z)
    drafts, u = s["drafts"].long(), s["uniforms"].double()
    some = drafts >= 0
    at = drafts.clamp(min=0)
    q = torch.ones(n, k, device="cuda", dtype=torch.float64)
    if case["slots"]:
        slots = _softmax(s["teacher"].double())
        q = torch.where(s["ids"].long() == at[:, :, None], slots, 0.0).sum(2)
    kept = some & (u[:, :k] * q < p[:, :k].gather(2, at[:, :, None])[:, :, 0])
    accepted = torch.cumprod(kept.long(), 1).sum(1)
    rows = torch.arange(n, device="cuda")
    w = p[rows, accepted]
    if k:
        row = accepted.clamp(max=k - 1)
        refused = (accepted < k) & some[rows, row]
        gone = torch.zeros_like(w)
        if case["slots"]:
            gone.scatter_add_(1, s["ids"][rows, row].long(), slots[rows, row])
        else:
            gone.scatter_(1, at[rows, row][:, None], 1.0)
        w = torch.where(refused[:, None], (w - gone).clamp(min=0.0), w)
    below = torch.cumsum(w, 1)
    chosen = (below <= u[:, k:] * below[:, -1:]).sum(1)
    tokens = torch.cat([drafts, torch.zeros_like(drafts[:, :1]) if k else chosen[:, None]], 1)
    place = torch.arange(k + 1, device="cuda")[None, :]
    tokens = torch.where(place == accepted[:, None], chosen[:, None], torch.where(place < accepted[:, None], tokens, -1))
    logp = torch.log(p.gather(2, tokens.clamp(min=0)[:, :, None])[:, :, 0])
    return tokens.int(), accepted.int(), torch.where(tokens >= 0, logp, 0.0).float()


def run(s):
    case = s["case"]
    op = case["op"]
    if own:
        import dciknn_cuda_amd as D
        if op in ("scan", "scantrain"):
            h, last = D.gated_scan(s["x"], s["gates"], s["state"], decay=case["decay"], lengths=s["lengths"], offsets=s["offsets"])
            if op == "scan":
                return h, last
            return (h.detach(), last.detach()) + torch.autograd.grad((h, last), s["leaves"], (s["dh"], s["dlast"]))
        if op == "norm":
            return D.grad_norm(s["grads"], scale=case["scale"])
        if op == "clip":
            norm = D.clip_grads(s["grads"], s["max_norm"], scale=case["scale"], out=s["out"])
            return norm, s["flat"]
        return D.verify_drafts(s["logits"], s["drafts"], s["uniforms"], s["ids"], s["teacher"], temperature=case["temperature"])
    with torch.no_grad():
        if op in ("scan", "scantrain"):
            return _plain_scan(s)
        if op == "verify":
            return _plain_verify(s)
        norm = torch.stack([(g.double() * g.double()).sum() for g in s["grads"]]).sum().sqrt() * case["scale"]
        if op == "norm":
            return norm.float()
        factor = (torch.clamp(s["max_norm"] / norm, max=1.0) * case["scale"]).float()
        for g, o in zip(s["grads"], s["out"] or s["grads"]):
            o.copy_(g.float() * factor)
        return norm.float(), s["flat"]


def work(case):
    size = BYTES[case["dtype"]]
    if case["op"] in ("scan", "scantrain"):
        n, d = case["batch"], case["dim"]
        cells = case["length"] * d * (1 if case["form"] == "packed" else n)
        gates = d if case["shared"] else cells
        states = n * d * 4
        if case["op"] == "scan":
            return {"bytes": (2 * cells + gates) * size + states * (1 + case["state"]), "flops": 10 * cells}
        return {"bytes": (4 * cells + 2 * gates) * size + states * (2 + 2 * case["state"]), "flops": 25 * cells}
    if case["op"] in ("norm", "clip"):
        cells = sum(math.prod(shape) for shape in _shapes(case))
        if case["op"] == "norm":
            return {"bytes": cells * size, "flops": 2 * cells}
        written = {"same": size, "f32": 4, "place": 0}[case["into"]]
        return {"bytes": cells * (size + written), "flops": 3 * cells}
    n, k, v = case["batch"], case["drafts"], case["vocab"]
    ids = 8 if case["ids64"] else 4
    return {"bytes": n * (k + 1) * (v * size + 12) + n * k * (ids + case["slots"] * (ids + 4)), "flops": 6 * n * (k + 1) * v}


def _exact_scan(s):
    """Token by token; sequences of a batch side by side, packed ones behind one another."""
    case = s["case"]
    n, t, d, decay = case["batch"], case["length"], case["dim"], case["decay"]
    x = s["x"].detach().double().reshape(-1, t, d)                       # [1 or n, t, d]
    g = s["gates"].detach().double()
    a = (g if decay else torch.sigmoid(g)).expand(s["x"].shape).reshape(x.shape)
    state = s["state"].detach().double() if case["state"] else torch.zeros(n, d, device="cuda", dtype=torch.float64)
    packed = case["form"] == "packed"
    bounds = s["offsets"].tolist() if packed else None
    lengths = s["lengths"].tolist() if s["lengths"] is not None else [t] * n
    h, before, last = torch.zeros_like(x), torch.zeros_like(x), state.clone()
    now = state.clone()
    first, end = {}, {}
    for i in range(n if packed else 0):
        if bounds[i + 1] > bounds[i]:
            first[bounds[i]], end[bounds[i + 1] - 1] = i, i
    alive = torch.tensor(lengths, device="cuda")[:, None]
    for j in range(t):
        if packed and j in first:
            now = state[first[j]][None]
        before[:, j] = now
        now = a[:, j] * now + x[:, j] if decay else torch.lerp(x[:, j], now, a[:, j])
        h[:, j] = now
        if packed and j in end:
            last[end[j]] = now[0]
    if not packed:
        rows = torch.arange(n, device="cuda")
        filled = alive[:, 0] > 0
        last = torch.where(filled[:, None], h[rows, (alive[:, 0] - 1).clamp(min=0)], state)
        if s["lengths"] is not None:
            h *= torch.arange(t, device="cuda")[None, :, None] < alive[:, :, None]
    if case["op"] == "scan":
        return h.reshape(s["x"].shape), last
    l = s["dh"].double().reshape(x.shape).clone()
    dlast = s["dlast"].double()
    dstate = dlast.clone()
    now = torch.zeros_like(now)
    for j in range(t - 1, -1, -1):
        if packed:
            now = (dlast[end[j]][None] if j in end else now) + l[:, j]
        else:
            now = torch.where(alive > j, torch.where(alive == j + 1, dlast, now) + l[:, j], 0.0)
        l[:, j] = now
        now = a[:, j] * now
        if packed and j in first:
            dstate[first[j]] = now[0]
    if not packed:
        dstate = torch.where(alive > 0, now, dlast)
    dx, dg = (l, l * before) if decay else (l * torch.sigmoid(-g).expand(s["x"].shape).reshape(x.shape), l * (before - x) * a * (1.0 - a))
    dg = dg.reshape(-1, d).sum(0) if case["shared"] else dg.reshape(s["x"].shape)
    return (h.reshape(s["x"].shape), last, dx.reshape(s["x"].shape), dg) + ((dstate,) if case["state"] else ())


def _exact_verify(s):
    """Sequence by sequence."""
    case = s["case"]
    k, v = case["drafts"], case["vocab"]
    drafts, u = s["drafts"].tolist(), s["uniforms"].double().tolist()
    tokens = torch.full((case["batch"], k + 1), -1, dtype=torch.int32)
    accepted, logps = torch.zeros(case["batch"], dtype=torch.int32), torch.zeros(case["batch"], k + 1, dtype=torch.float64)
    for b in range(case["batch"]):
        for i in range(k + 1):
            logp = torch.log_softmax(s["logits"][b, i].double() / case["temperature"], 0)
            p = logp.exp()
            if i == k or drafts[b][i] < 0:
                break
            q = torch.zeros(v, dtype=torch.float64, device="cuda")
            if case["slots"]:
                q.index_add_(0, s["ids"][b, i].long(), torch.softmax(s["teacher"][b, i].double(), 0))
            else:
                q[drafts[b][i]] = 1.0
            if not u[b][i] * q[drafts[b][i]].item() < p[drafts[b][i]].item():
                p = (p - q).clamp(min=0.0)
                break
            tokens[b, i], logps[b, i] = drafts[b][i], logp[drafts[b][i]].item()
            accepted[b] += 1
        sums = torch.cumsum(p, 0)
        chosen = torch.searchsorted(sums, sums[-1:] * u[b][k], right=True).item()
        tokens[b, i], logps[b, i] = chosen, logp[chosen].item()
    return tokens.cuda(), accepted.cuda(), logps.cuda()


def exact(case, seed):
    """The definitions in 64 bits."""
    s = prepare(case, seed)
    if case["op"] in ("scan", "scantrain"):
        return _exact_scan(s)
    if case["op"] == "verify":
        return _exact_verify(s)
    squares = torch.tensor([torch.linalg.vector_norm(g.double()).item() ** 2 for g in s["grads"]], dtype=torch.float64)
    scale = s["case"]["scale"]
    norm = math.sqrt(math.fsum(squares.tolist())) * scale
    if case["op"] == "norm":
        return torch.tensor(norm, dtype=torch.float64, device="cuda")
    factor = min(1.0, s["max_norm"] / norm) * scale
    return torch.tensor(norm, dtype=torch.float64, device="cuda"), torch.cat([g.double().flatten() for g in s["grads"]]) * factor
