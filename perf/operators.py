"""What the time of the token operators is measured on.

A case is one call, or a call and its gradient, that a program makes which trains or serves
a model on rows and neighbours that `DCI` indexes and finds:

  embed       rows of a table by ids, times a factor (`embed`)
  embedgrad   the gradient of that by the table, summed over the tokens of each row (`embed_grad`)
  logprobs    log probabilities of given tokens, entropies, best alternatives (`token_logprobs`)
  logtrain    the same without alternatives, and the gradient by the logits
  distill     the loss against a teacher's top logits and its gradient, as autograd asks for
              them: one after the other (`distill_loss`)
  distillstep loss and gradient by one call (`distill_step`)

With `own` false they are computed in their plain form, in 32 bits, by elementary torch
operations.  Ids of natural text are spread evenly over their logarithm (a few are most of the
tokens); ids of neighbours are spread evenly over the rows.
"""
import torch

own = False

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
BYTES = {"f32": 4, "bf16": 2, "f16": 2}


def _case(name, op, n, v, dim=0, k=0, dtype="bf16", spread="text", ids64=True, scale=1.0, masked=False):
    """n tokens; v rows of the table or entries of the vocabulary; dim: a row's length; k: top
    alternatives or the teacher's slots; scale: the lookup's factor or the temperature;
    masked: in every second row of logits all but some hundred tokens are ruled out by -inf."""
    c = dict(op=op, n=n, v=v, dim=dim, k=k, dtype=dtype, spread=spread, ids64=ids64, scale=scale, masked=masked)
    if name:
        c["name"] = name
    return c


def listed():
    return [
        # One step of a server: the tokens of 32 sequences.
        _case("embed-step", "embed", 32, 32_000, 4096, scale=64.0),
        # A batch of long prompts.
        _case("embed-prompt", "embed", 32_768, 131_072, 4096, scale=64.0),
        # The neighbours of 10k queries in the benchmark's table, taken by the ids of DCI.query.
        _case("embed-neighbours", "embed", 100_000, 1_000_000, 128, dtype="f32", spread="even", ids64=False),
        # Fine-tuning on the table of the reference's example: rows of 400 bytes.
        _case("grad-small", "embedgrad", 1000, 3000, 100, dtype="f32", spread="even", ids64=False),
        # A training step's tokens: the commonest is a tenth of them.
        _case("grad-train", "embedgrad", 65_536, 50_001, 2048, scale=45.25),
        # The gradient by the benchmark's table of what the neighbours' rows were used for.
        _case("grad-neighbours", "embedgrad", 100_000, 1_000_000, 128, dtype="f32", spread="even", ids64=False),
        # A server's step: four sequences' tokens with 20 alternatives, some under a grammar.
        _case("logprobs-step", "logprobs", 4, 131_072, k=20, masked=True),
        # Scoring of given text; rows of odd length.
        _case("logprobs-score", "logprobs", 4096, 50_001, k=5, dtype="f16"),
        # Policy gradients with an entropy bonus, logits in 32 bits.
        _case("logprobs-train", "logtrain", 8192, 32_000, dtype="f32", scale=0.7),
        # The reference's example as a retrieval head: 10 neighbours among 3000 rows, 500 queries.
        _case("distill-small", "distill", 500, 3000, k=10, dtype="f32", spread="even", ids64=False),
        # Odd sizes: a hundred neighbours, a vocabulary of odd length.
        _case("distill-ragged", "distillstep", 1001, 100_003, k=100, dtype="f16", ids64=False, scale=2.0),
        # A training step.
        _case("distill-train", "distillstep", 8192, 131_072, k=64),
    ]


def _spread(rng, lo, hi):
    """A whole number in [lo, hi], even over its logarithm."""
    return min(hi, max(lo, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    op = rng.choice(["embed", "embed", "embedgrad", "embedgrad", "logprobs", "logprobs", "logtrain", "distill", "distillstep", "distillstep"])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    spread = rng.choice(["text", "text", "even"])
    ids64 = rng.random() < 0.6
    if op in ("embed", "embedgrad"):
        v, dim = _spread(rng, 1000, 1_000_000), _spread(rng, 16, 8192)
        if rng.random() < 0.7:                     # most rows are whole 16-byte words
            dim = (dim + 7) // 8 * 8
        n = _spread(rng, 1, 131_072)
        v = min(v, 256_000_000 // dim)             # no table above those listed by much
        n = max(1, min(n, 134_217_728 // dim))
        return _case(None, op, n, v, dim, 0, dtype, spread, ids64, rng.choice([1.0, dim ** 0.5, 0.5]))
    v, n = _spread(rng, 1000, 262_144), _spread(rng, 1, 16_384)
    if rng.random() < 0.6:                         # most vocabularies are padded to whole lines
        v = (v + 63) // 64 * 64
    n = max(1, min(n, (1 << 29) // v))
    k = _spread(rng, 1, 32) if op == "logprobs" else 0 if op == "logtrain" else _spread(rng, 4, 128)
    masked = op == "logprobs" and rng.random() < 0.3
    return _case(None, op, n, v, 0, k, dtype, spread, ids64, rng.choice([1.0, 1.0, 0.7, 2.0]), masked)


def _ids(case, shape, gen, empty):
    """Ids below case["v"], a share `empty` of them -1."""
    u = torch.rand(shape, generator=gen, device="cuda", dtype=torch.float64)
    v = case["v"]
    ids = (v * u if case["spread"] == "even" else float(v) ** u - 1.0).long().clamp_(0, v - 1)
    if empty:
        ids[torch.rand(shape, generator=gen, device="cuda") < empty] = -1
    return ids if case["ids64"] else ids.int()


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    n, v, dim, k, dtype = case["n"], case["v"], case["dim"], case["k"], TYPES[case["dtype"]]
    s = dict(case=case)

    def randn(*shape):
        return torch.randn(*shape, generator=gen, device="cuda")

    if case["op"] in ("embed", "embedgrad"):
        s["ids"] = _ids(case, (n,), gen, 0.02 if case["spread"] == "text" else 0.0)
        if case["op"] == "embed":
            s["table"] = torch.empty(v, dim, device="cuda", dtype=dtype).normal_(0.0, 0.02, generator=gen)
        else:
            s["grad"] = (randn(n, dim) * 0.01).to(dtype)
        return s
    z = torch.empty(n, v, device="cuda", dtype=torch.float32).normal_(0.0, 2.5, generator=gen)
    # the right token is mostly among the likely ones
    s["targets"] = _ids(case, (n,), gen, 0.02)
    right = s["targets"].long().clamp(min=0)
    rows = torch.arange(n, device="cuda")
    z[rows, right] += 12.0 * torch.rand(n, generator=gen, device="cuda")
    if case["masked"]:
        keep = torch.rand(n, v, generator=gen, device="cuda") < min(0.5, 200.0 / v)
        keep[1::2] = True
        keep[rows, right] = True
        z.masked_fill_(~keep, float("-inf"))
    s["logits"] = z.to(dtype)
    # a mean over the tokens; with gradients in f16 the loss is scaled up, here by their number
    share = 1.0 if case["dtype"] == "f16" else 1.0 / n
    if case["op"] == "logtrain":
        s["dlogprobs"], s["dentropy"] = randn(n) * share, torch.full((n,), -0.01 * share, device="cuda")
    if case["op"].startswith("distill"):
        # neighbours of a query: distances in ascending order, the next tokens of some the same;
        # the last slots of some rows are empty
        s["teacher_ids"] = _ids(case, (n, k), gen, 0.0)
        s["teacher"] = -torch.sort(6.0 * torch.rand(n, k, generator=gen, device="cuda"), dim=1).values
        filled = 1 + (k * 4 * torch.rand(n, 1, generator=gen, device="cuda")).int()
        gone = torch.arange(k, device="cuda")[None, :] >= filled
        s["teacher_ids"].masked_fill_(gone, -1)
        s["teacher"].masked_fill_(gone, float("-inf"))
        s["weights"] = torch.rand(n, generator=gen, device="cuda") * share
    if case["op"] in ("logtrain", "distill"):
        s["logits"].requires_grad_()
    return s


def _top(z, k):
    """The k largest of each row, ties to the lowest index: one whole number orders both."""
    bits = (z + 0.0).view(torch.int32)
    order = torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits).long()
    back = torch.arange(z.shape[1] - 1, -1, -1, device=z.device)
    best = torch.topk((order << 32) | back, k, dim=1).values
    return z.shape[1] - 1 - (best & 0xFFFFFFFF)


def _plain(s):
    case = s["case"]
    op, v, scale, dtype = case["op"], case["v"], case["scale"], TYPES[case["dtype"]]
    if op == "embed":
        ids = s["ids"].long()
        rows = s["table"][ids.clamp(min=0)].float() * scale
        return (rows * (ids >= 0)[:, None]).to(dtype)
    if op == "embedgrad":
        ids = s["ids"].long()
        rows = s["grad"].float() * (scale * (ids >= 0).float())[:, None]
        return torch.zeros(v, case["dim"], device="cuda").index_add_(0, ids.clamp(min=0), rows).to(dtype)
    z = s["logits"].detach().float()
    x = (z - z.max(dim=1, keepdim=True).values) / scale
    e = torch.exp(x)
    total = e.sum(dim=1, keepdim=True)
    lse = torch.log(total)
    if op in ("logprobs", "logtrain"):
        t = s["targets"].long()[:, None]
        some = t >= 0
        logp = torch.where(some, x.gather(1, t.clamp(min=0)) - lse, 0.0)
        entropy = lse - (e * x.clamp(min=-200.0)).sum(dim=1, keepdim=True) / total
        if op == "logprobs":
            ids = _top(z, case["k"])
            return logp[:, 0], entropy[:, 0], ids.int(), x.gather(1, ids) - lse
        p = e / total
        g, h = s["dlogprobs"][:, None], s["dentropy"][:, None]
        dz = -p * (torch.where(some, g, 0.0) + h * (x.clamp(min=-200.0) - lse + entropy))
        dz = dz.scatter_add(1, t.clamp(min=0), torch.where(some, g, 0.0)) / scale
        return logp[:, 0], entropy[:, 0], dz.to(dtype)
    ids, teacher = s["teacher_ids"].long(), s["teacher"]
    some = (ids >= 0) & (teacher > float("-inf"))
    ids = ids.clamp(min=0)
    y = (torch.where(some, teacher, float("-inf")) - teacher.max(dim=1, keepdim=True).values) / scale
    f = torch.exp(y)
    q = f / f.sum(dim=1, keepdim=True)
    logq = y - torch.log(f.sum(dim=1, keepdim=True))
    loss = torch.where(some, q * (logq - (x.gather(1, ids) - lse)), 0.0).sum(dim=1)
    dz = (e / total).scatter_add(1, ids, -q) * (s["weights"][:, None] / scale)
    return loss, dz.to(dtype)


def run(s):
    if not own:
        with torch.no_grad():
            return _plain(s)
    import dciknn_cuda_amd as D
    case = s["case"]
    op, scale = case["op"], case["scale"]
    if op == "embed":
        return D.embed(s["table"], s["ids"], scale)
    if op == "embedgrad":
        return D.embed_grad(s["grad"], s["ids"], case["v"], scale)
    if op == "logprobs":
        return D.token_logprobs(s["logits"], s["targets"], top=case["k"], temperature=scale)
    if op == "logtrain":
        logp, entropy = D.token_logprobs(s["logits"], s["targets"], temperature=scale)
        dz, = torch.autograd.grad((logp, entropy), s["logits"], (s["dlogprobs"], s["dentropy"]))
        return logp.detach(), entropy.detach(), dz
    if op == "distill":
        loss = D.distill_loss(s["logits"], s["teacher_ids"], s["teacher"], temperature=scale)
        dz, = torch.autograd.grad(loss, s["logits"], s["weights"])
        return loss.detach(), dz
    return D.distill_step(s["logits"], s["teacher_ids"], s["teacher"], s["weights"], temperature=scale)


def _distinct(case):
    """How many rows the lookups of a case are expected to reach."""
    i = torch.arange(case["v"], dtype=torch.float64)
    chance = torch.log1p(1.0 / (i + 1.0)) / torch.log(torch.tensor(float(case["v"])))
    chance = chance if case["spread"] == "text" else torch.full_like(i, 1.0 / case["v"])
    return float((1.0 - torch.exp(-case["n"] * chance)).sum())


def work(case):
    n, v, dim, k, size = case["n"], case["v"], case["dim"], case["k"], BYTES[case["dtype"]]
    idsize = 8 if case["ids64"] else 4
    if case["op"] == "embed":
        # each row that is looked up is read once at least
        return {"bytes": n * idsize + (n + _distinct(case)) * dim * size, "flops": n * dim}
    if case["op"] == "embedgrad":
        return {"bytes": n * idsize + (n + v) * dim * size, "flops": 2 * n * dim}
    if case["op"] == "logprobs":
        return {"bytes": n * v * size + n * (idsize + 8 + 8 * k), "flops": 5 * n * v}
    if case["op"] == "logtrain":
        return {"bytes": 2 * n * v * size + n * (idsize + 16), "flops": 10 * n * v}
    return {"bytes": 2 * n * v * size + n * (k * (idsize + 4) + 8), "flops": 6 * n * v}


def exact(case, seed):
    """The definitions in 64 bits, row by row where the rows are independent."""
    s = prepare(case, seed)
    op, n, v, T = case["op"], case["n"], case["v"], case["scale"]
    if op == "embed":
        got = torch.zeros(n, case["dim"], dtype=torch.float64, device="cuda")
        filled = torch.nonzero(s["ids"] >= 0)[:, 0]
        got[filled] = s["table"].index_select(0, s["ids"][filled].long()).double().mul_(T)
        return got
    if op == "embedgrad":
        # differences of running sums over the tokens, ordered by their row, in slices of the columns
        ids, order = torch.sort(s["ids"].long(), stable=True)
        ends = torch.searchsorted(ids, torch.arange(-1, v, device="cuda"), right=True)
        got = torch.empty(v, case["dim"], dtype=torch.float64, device="cuda")
        for c in range(0, case["dim"], 256):
            sums = torch.zeros(n + 1, min(256, case["dim"] - c), dtype=torch.float64, device="cuda")
            torch.cumsum(s["grad"][order, c:c + 256].double(), 0, out=sums[1:])
            got[:, c:c + 256] = (sums[ends[1:]] - sums[ends[:-1]]) * T
        return got
    step, parts = max(1, (1 << 27) // v), []
    for a in range(0, n, step):
        z = s["logits"][a:a + step].detach().double()
        logp = torch.log_softmax(z / T, dim=1)
        p = torch.exp(logp)
        if op in ("logprobs", "logtrain"):
            t = s["targets"][a:a + step].long()
            given = torch.nonzero(t >= 0)[:, 0]
            lp = torch.zeros(z.shape[0], dtype=torch.float64, device="cuda")
            lp[given] = logp[given, t[given]]
            plogp = torch.where(p > 0, p * logp, 0.0)
            entropy = -plogp.sum(1)
            if op == "logprobs":
                ids = torch.sort(z, dim=1, descending=True, stable=True).indices[:, :case["k"]]
                parts.append((lp, entropy, ids.int(), logp.gather(1, ids)))
                continue
            g, h = s["dlogprobs"][a:a + step].double(), s["dentropy"][a:a + step].double()
            dz = -h[:, None] * (plogp + p * entropy[:, None])
            dz[given] -= g[given, None] * p[given]
            dz[given, t[given]] += g[given]
            parts.append((lp, entropy, dz / T))
            continue
        ids = s["teacher_ids"][a:a + step].long()
        some = ids >= 0
        logq = torch.log_softmax(s["teacher"][a:a + step].double().masked_fill(~some, float("-inf")) / T, dim=1)
        q = torch.where(some, torch.exp(logq), 0.0)
        at = ids.clamp(min=0)
        loss = torch.where(some & (q > 0), q * (logq - logp.gather(1, at)), 0.0).sum(1)
        p.scatter_add_(1, at, -q)
        parts.append((loss, p * (s["weights"][a:a + step].double() / T)[:, None]))
    return tuple(torch.cat([part[i] for part in parts]) for i in range(len(parts[0])))
