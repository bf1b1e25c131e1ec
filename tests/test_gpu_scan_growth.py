"""The recurrence with decays beyond 1, whose product over a tile is beyond 32 bits while the states themselves are not, against 64 bits."""
import numpy as np
import pytest
import torch

import recurrent_oracles as O
from test_gpu_scan import TYPES, VIEWS, near

pytestmark = pytest.mark.gpu


def wandering(rows, length, dim, span, steps, seed):
    """(decays, 2 to the what of their product up to and including each token): the product goes up and down within 2^-span and 2^span, by 2^steps[t]
    about a token."""
    rng = np.random.default_rng(seed)
    a, level = np.empty((rows, length, dim)), np.empty((rows, length, dim))
    now = np.zeros((rows, dim))
    for t in range(length):
        by = rng.normal(size=(rows, dim)) * steps[t]
        by = np.where(np.abs(now + by) > span, -by, by)
        by = np.clip(now + by, -span, span) - now
        a[:, t] = np.float32(2.0 ** by) * np.where(rng.random((rows, dim)) < 0.3, -1.0, 1.0)
        now = now + by
        level[:, t] = now
    return a, level


def check(gpu, x, gates, state, dh, dlast, dtype, lengths=None, offsets=None, only=slice(None)):
    """All of [rows, length, dim], gates also [dim]; float64 arrays that `dtype` rounds."""
    rows, length, dim = x.shape
    to = lambda v: torch.from_numpy(np.ascontiguousarray(v)).to(TYPES[dtype])         # noqa: E731
    x, gates, dh = to(x), to(gates), to(dh)
    n = rows if offsets is None else len(offsets) - 1
    s = torch.zeros(n, dim) if state is None else torch.from_numpy(state).float()
    dl = torch.from_numpy(dlast).float()
    num = lambda t: t.double().numpy()                                               # noqa: E731
    shared = gates.dim() == 1
    seqs = O.sequences_of(rows, length, lengths, offsets)
    if offsets is None:
        seqs = seqs[only]
    picked = range(n)[only] if offsets is None else range(n)
    full = np.broadcast_to(num(gates), x.shape)
    h, last, _, err, last_err = O.gated_scan(num(x), full, num(s)[picked], seqs, True)
    dx, dg, ds, ex, eg, es = O.gated_scan_grad(num(x), full, num(s)[picked], seqs, True, num(dh), num(dl)[picked])
    # (of the inputs: nothing that is held in 32 bits is beyond them)
    assert max(np.abs(v).max() for v in (h, dx, dg)) < 2.0 ** 120
    flat = (lambda t: t[0]) if offsets is not None else (lambda t: t)
    leaves = [flat(x).cuda().requires_grad_(), (gates if shared else flat(gates)).cuda().requires_grad_()] + ([] if state is None else [s.cuda().requires_grad_()])
    kw = dict(decay=True, lengths=None if lengths is None else torch.tensor(lengths).cuda(), offsets=None if offsets is None else torch.tensor(offsets).cuda())
    first = leaves[2] if state is not None else None
    with torch.no_grad():
        plain = gpu.gated_scan(leaves[0], leaves[1], first, **kw)
    out = gpu.gated_scan(leaves[0], leaves[1], first, **kw)
    got = torch.autograd.grad(out, leaves, (flat(dh).cuda(), dl.cuda()))
    pick = lambda t: t.reshape(x.shape)[only] if offsets is None else t.reshape(x.shape)      # noqa: E731
    rows_of = (lambda v: v[only]) if offsets is None else (lambda v: v)
    for one in (plain, out):
        near(pick(one[0]), rows_of(h), rows_of(err), dtype, "h")
        near(one[1][only] if offsets is None else one[1], last, last_err, "f32", "last")
    near(pick(got[0]), rows_of(dx), rows_of(ex), dtype, "dx")
    if shared:
        near(got[1], dg.sum((0, 1)), eg.sum((0, 1)) + 40.0 * np.abs(dg).sum((0, 1)), dtype, "dgates")
    else:
        near(pick(got[1]), rows_of(dg), rows_of(eg), dtype, "dgates")
    if state is not None:
        near(got[2][only] if offsets is None else got[2], ds, es, "f32", "dstate")


def scaled(rng, level, seqs):
    """x, states, and gradients for h and the last states, of the sizes at which all products are about 1."""
    x, dh = 2.0 ** level * rng.normal(size=level.shape), 2.0 ** -level * rng.normal(size=level.shape)
    ahead = [np.exp2(level[r, a - 1] if a else np.zeros(level.shape[2])) for r, a, _ in seqs]
    behind = [np.exp2(-level[r, b - 1] if b else np.zeros(level.shape[2])) for r, _, b in seqs]
    return x, np.stack(ahead) * rng.normal(size=(len(seqs), level.shape[2])), dh, np.stack(behind) * rng.normal(size=(len(seqs), level.shape[2]))


# (a stretch that hardly changes, one that changes much, by turns)
CALM = lambda t: 4.0 if t // 300 % 2 else 0.02          # noqa: E731


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("size", [(3, 700, 24), (2, 1000, 5), (1, 1300, 33), (4, 129, 130), (7, 40, 16), (5, 65, 8), (3, 17, 3)], ids=str)
@pytest.mark.parametrize("span, step", [(40.0, CALM), (60.0, lambda t: 25.0), (40.0, lambda t: 0.5)], ids=["stretches", "steep", "mild"])
def test_products_that_wander(gpu, size, span, step, dtype):
    rng = np.random.default_rng(size[1])
    a, level = wandering(*size, span, [step(t) for t in range(size[1])], size[2])
    x, state, dh, dlast = scaled(rng, level, O.sequences_of(size[0], size[1]))
    check(gpu, x, a, state, dh, dlast, dtype)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("offsets", [[0, 900], [3, 10, 10, 140, 700, 880], [0, 128, 256, 256, 600, 900], list(range(0, 901, 25))], ids=lambda v: str(v)[:20])
def test_packed(gpu, offsets, dtype):
    rng = np.random.default_rng(1)
    a, level = wandering(1, 900, 18, 40.0, [CALM(t) for t in range(900)], 2)
    x, state, dh, dlast = scaled(rng, level, O.sequences_of(1, 900, offsets=offsets))
    check(gpu, x, a, state, dh, dlast, dtype, offsets=offsets)


@pytest.mark.parametrize("length, lengths", [(700, [513, 3, 0, 700]), (33, [33, 0, 17, 1, 32])])
def test_lengths(gpu, length, lengths):
    rng = np.random.default_rng(3)
    a, level = wandering(len(lengths), length, 20, 40.0, [CALM(t + 300) for t in range(length)], 4)
    x, state, dh, dlast = scaled(rng, level, O.sequences_of(len(lengths), length, lengths))
    # (what stands behind a sequence's end is not looked at)
    for row, n in enumerate(lengths):
        x[row, n:], dh[row, n:], a[row, n:] = np.nan, np.nan, np.inf
    full = lambda v: np.where(np.isfinite(v), v, 0.0)                                # noqa: E731
    check(gpu, x, a, state, full(dh), dlast, "f32", lengths=lengths)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("offsets", [None, [0, 26_000], [0, 9_000, 9_001, 26_000]], ids=["one", "offsets", "three"])
def test_a_long_chain(gpu, offsets, dtype):
    """Tiles whose maps are formed by a launch of their own."""
    rng = np.random.default_rng(5)
    span = 8.0 if dtype == "f16" else 40.0
    a, level = wandering(1, 26_000, 40, span, [(1.5 if dtype == "f16" else 3.0) if 4000 < t < 5000 or 20_000 < t < 20_100 else 0.01 for t in range(26_000)], 6)
    a = np.clip(a, -60_000.0, 60_000.0)
    x, state, dh, dlast = scaled(rng, level, O.sequences_of(1, 26_000, offsets=offsets))
    quiet = np.minimum(1.0, np.arange(26_000) % 50 == 0)[None, :, None]              # (sums that stay within the type)
    check(gpu, x * quiet, a, state, dh * quiet, dlast, dtype, offsets=offsets)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("shared", [False, True])
@pytest.mark.parametrize("size", [(3, 600, 24), (1, 700, 5), (6, 64, 16), (6, 30, 9), (1, 26_000, 24)], ids=str)
def test_growth_of_nothing(gpu, size, shared, dtype):
    """States and gradients that are 0 stay 0 however large the factors' product is."""
    rng = np.random.default_rng(8)
    rows, length, dim = size
    few = min(length // 3, 15)
    a = np.full((dim,) if shared else size, 2.0 if length > 100 else 500.0)
    x, dh = np.zeros(size), np.zeros(size)
    x[:, -few:], dh[:, :few] = rng.normal(size=(rows, few, dim)), rng.normal(size=(rows, few, dim))
    if length <= 100:
        x[:, :-1], dh[:, 1:] = 0.0, 0.0
    check(gpu, x, a, None, dh, np.zeros((rows, dim)), dtype)


def test_a_little_beyond_1(gpu):
    """Decays around 1, as those that are learnt may be."""
    rng = np.random.default_rng(9)
    for size in ((2, 1000, 24), (1, 26_000, 24)):
        a = 1.0 + 0.03 * rng.normal(size=size)
        a[:, ::40] = 0.3
        check(gpu, rng.normal(size=size), a, rng.normal(size=(size[0], 24)), rng.normal(size=size), rng.normal(size=(size[0], 24)), "f32")


@pytest.mark.parametrize("rows", [2, 256])
def test_many_rows_as_few(gpu, rows):
    """By a thread a piece of a row, or by tiles: what is returned for a row depends on its values alone."""
    rng = np.random.default_rng(10)
    length, dim = 140, 2048
    a, level = wandering(2, length, 16, 40.0, [3.0] * length, 11)
    a, level = np.tile(a, (1, 1, dim // 16)), np.tile(level, (1, 1, dim // 16))
    x, state, dh, dlast = scaled(rng, level, O.sequences_of(2, length))
    many = lambda v: np.concatenate([v] * (rows // 2))                               # noqa: E731
    check(gpu, many(x), many(a), many(state), many(dh), many(dlast), "bf16", only=slice(0, 2))


@pytest.mark.parametrize("view", VIEWS)
@pytest.mark.parametrize("size", [(3, 300, 18), (2, 26_000, 16)], ids=str)
@pytest.mark.parametrize("shared", [False, True])
def test_strides(gpu, size, shared, view):
    """Where tokens stand changes no bit."""
    rng = np.random.default_rng(14)
    a, level = wandering(*size, 40.0, [3.0 if t % 5000 < 200 else 0.01 for t in range(size[1])], 15)
    x, state, dh, dlast = (torch.from_numpy(v).float().cuda() for v in scaled(rng, level, O.sequences_of(size[0], size[1])))
    a = torch.from_numpy(a).float().cuda()
    if shared:
        a = torch.full((size[2],), 1.8, device="cuda")
        x[:, :-20], dh[:, 20:], state, dlast = 0.0, 0.0, None, torch.zeros_like(dlast)
    results = []
    for of in (lambda t: t, VIEWS[view]):
        leaves = [of(x).detach().requires_grad_(), (a if shared else of(a)).detach().requires_grad_()] + ([] if shared else [state.detach().requires_grad_()])
        out = gpu.gated_scan(leaves[0], leaves[1], None if shared else leaves[2], decay=True)
        results.append(list(out) + list(torch.autograd.grad(out, leaves, (of(dh), dlast))))
    assert all(torch.equal(p, q) for p, q in zip(*results))
    assert all(bool(p.isfinite().all()) for p in results[0])


def test_decays_that_are_not_finite(gpu):
    """They leave nothing finite behind them in their channel, and touch no other."""
    x = torch.randn(2, 500, 16, generator=torch.Generator().manual_seed(12))
    a = torch.full((2, 500, 16), 0.9)
    a[0, 137, 3], a[1, 300, 5], a[1, 0, 7] = float("inf"), float("nan"), float("-inf")
    h, last = gpu.gated_scan(x.cuda(), a.cuda(), decay=True)
    fine = torch.ones(2, 500, 16, dtype=torch.bool)
    fine[0, 137:, 3] = fine[1, 300:, 5] = fine[1, 0:, 7] = False
    assert torch.equal(h.isfinite().cpu(), fine) and torch.equal(last.isfinite().cpu(), fine[:, -1])


def test_recorded_and_replayed(gpu):
    rng = np.random.default_rng(13)
    static = [torch.zeros(1, 26_000, 40, device="cuda") for _ in range(2)]
    graph = None
    for turn in range(4):
        a, level = wandering(1, 26_000, 40, 40.0, [3.0 if turn % 2 and t > 25_000 else 0.02 for t in range(26_000)], turn)
        static[0].copy_(torch.from_numpy(2.0 ** level * rng.normal(size=level.shape)))
        static[1].copy_(torch.from_numpy(a))
        want = gpu.gated_scan(*static, decay=True)
        if graph is None:
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                got = gpu.gated_scan(*static, decay=True)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1]) and bool(got[0].isfinite().all()), turn
