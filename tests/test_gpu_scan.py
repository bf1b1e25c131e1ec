"""The gated recurrence and its gradient against 64 bits, at the lengths, strides and values where they can go wrong."""
import numpy as np
import pytest
import torch

import recurrent_oracles as O

pytestmark = pytest.mark.gpu
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
# the least a type resolves, half a step of it
TINY = {"f32": 2.0 ** -126, "f16": 2.0 ** -25, "bf16": 2.0 ** -126}


def near(got, want, err, dtype, what):
    """`err` in units of half a step of 32 bits, and one rounding to `dtype`."""
    got = got.detach().double().cpu().numpy()
    half = torch.finfo(TYPES[dtype]).eps / 2
    bound = O.STEP * err * (1 + 2 * half) + half * np.abs(want) + TINY[dtype]
    # a value that may be beyond the type's largest rounds to infinity
    beyond = np.isinf(got) & (got * want > 0) & (np.abs(want) + bound > torch.finfo(TYPES[dtype]).max)
    worst = np.where(beyond, 0.0, np.abs(got - want) - bound)
    assert got.shape == want.shape and (worst <= 0).all(), "%s: off by %g where %g is allowed" % (
        what, np.abs(got - want).flat[np.argmax(worst)], bound.flat[np.argmax(worst)])


def inputs(rows, length, dim, dtype, decay, shared, packed=0, seed=0, state=True):
    g = torch.Generator().manual_seed(seed)
    shape = (length, dim) if packed else (rows, length, dim)
    x = torch.randn(shape, generator=g).to(TYPES[dtype])
    gates = torch.randn((dim,) if shared else shape, generator=g)
    gates = ((gates * 0.6).clamp(-1, 1) if decay else 1.0 + 3.0 * gates).to(TYPES[dtype])
    n = packed or rows
    s = torch.randn(n, dim, generator=g) if state else None
    dh, dlast = torch.randn(shape, generator=g).to(TYPES[dtype]), torch.randn(n, dim, generator=g)
    return x, gates, s, dh, dlast


def check(gpu, rows, length, dim, dtype, decay=False, shared=False, lengths=None, offsets=None, state=True, wide=False, seed=0, view=lambda t: t,
          grad=True):
    packed = 0 if offsets is None else len(offsets) - 1
    x, gates, s, dh, dlast = inputs(rows, length, dim, dtype, decay, shared, packed, seed, state)
    n = packed or rows
    ids = torch.int64 if wide else torch.int32
    dev = lambda t: None if t is None else t.cuda()                                   # noqa: E731
    kw = dict(decay=decay, lengths=dev(None if lengths is None else torch.tensor(lengths, dtype=ids)),
              offsets=dev(None if offsets is None else torch.tensor(offsets, dtype=ids)))
    flat = lambda t: t.double().numpy().reshape(1 if packed else rows, length, dim)   # noqa: E731
    full = gates.expand(x.shape) if shared else gates
    seqs = O.sequences_of(rows, length, lengths, offsets)
    s64 = np.zeros((n, dim)) if s is None else s.double().numpy()
    h, last, _, err, last_err = O.gated_scan(flat(x), flat(full), s64, seqs, decay)
    inside = np.zeros((1 if packed else rows, length, 1), bool)
    for row, lo, hi in seqs:
        inside[row, lo:hi] = True
    xd, gd = view(x.cuda()), gates.cuda() if shared else view(gates.cuda())
    got_h, got_last = gpu.gated_scan(xd, gd, dev(s), **kw)
    assert got_h.dtype == x.dtype and got_last.dtype == torch.float32 and got_h.shape == x.shape
    near(got_h.reshape(h.shape), h, err, dtype, "h")
    near(got_last, last, last_err, "f32", "last")
    assert not got_h.reshape(h.shape).float().cpu().numpy()[~np.broadcast_to(inside, h.shape)].any()
    if not grad:
        return
    leaves = [xd.detach().requires_grad_(), gd.detach().requires_grad_()] + ([dev(s).requires_grad_()] if state else [])
    out_h, out_last = gpu.gated_scan(leaves[0], leaves[1], leaves[2] if state else None, **kw)
    near(out_h.reshape(h.shape), h, err, dtype, "h of the call with gradients")
    near(out_last, last, last_err, "f32", "last of the call with gradients")
    got = torch.autograd.grad((out_h, out_last), leaves, (dh.cuda(), dlast.cuda()))
    dx, dg, ds, ex, eg, es = O.gated_scan_grad(flat(x), flat(full), s64, seqs, decay, flat(dh), dlast.double().numpy())
    near(got[0].reshape(dx.shape), dx, ex, dtype, "dx")
    if shared:
        # a sum of up to 36 terms in a tile's 32 bits
        near(got[1], dg.sum((0, 1)), eg.sum((0, 1)) + 40.0 * np.abs(dg).sum((0, 1)), dtype, "dgates")
    else:
        near(got[1].reshape(dg.shape), dg, eg, dtype, "dgates")
    if state:
        near(got[2], ds, es, "f32", "dstate")


SIZES = [(1, 1, 1), (3, 1, 64), (5, 16, 9), (2, 17, 33), (4, 64, 40), (3, 65, 16), (9, 5, 7), (2, 127, 8), (2, 128, 130), (1, 129, 257), (2, 300, 5), (3, 1000, 24)]


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("decay", [False, True])
@pytest.mark.parametrize("shared", [False, True])
@pytest.mark.parametrize("size", SIZES, ids=str)
def test_batch(gpu, size, shared, decay, dtype):
    check(gpu, *size, dtype, decay, shared, state=size[0] != 2)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("shared", [False, True])
@pytest.mark.parametrize("length, lengths", [(1, [1, 0]), (9, [0, 9, 4, 1, -3, 99]), (40, [40, 0, 17, 39, 1]), (200, [128, 129, 0, 200, 127, 1]), (700, [513, 3, 700])])
def test_lengths(gpu, length, lengths, shared, dtype):
    check(gpu, len(lengths), length, 20, dtype, False, shared, lengths=lengths, wide=shared)


PACKED = [(1, [0, 1]), (5, [0, 0, 5, 5]), (130, [0, 128, 130]), (300, [3, 10, 10, 140, 270]), (256, [0, 128, 128, 128, 256]), (900, [0, 1, 2, 3, 400, 401, 899, 900]),
          (500, list(range(0, 501, 1))), (700, [0] + [650] * 300 + [700]), (400, [400, 400]), (300, [-5, 7, 1000]), (64, [0] * 70 + [64])]


@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("decay", [False, True])
@pytest.mark.parametrize("tokens, offsets", PACKED, ids=lambda v: str(v)[:20])
def test_packed(gpu, tokens, offsets, decay, dtype):
    check(gpu, 1, tokens, 18, dtype, decay, offsets=offsets, wide=decay, shared=dtype == "f16" and decay)


def test_one_sequence_of_tokens(gpu):
    """[tokens, dim] without offsets."""
    x, gates, s, _, _ = inputs(1, 260, 12, "f32", False, False)
    a = gpu.gated_scan(x[0].cuda(), gates[0].cuda(), s.cuda())
    b = gpu.gated_scan(x.cuda(), gates.cuda(), s.cuda())
    assert torch.equal(a[0], b[0][0]) and torch.equal(a[1], b[1])


VIEWS = {
    "time first": lambda t: t.transpose(0, 1).contiguous().transpose(0, 1),
    "part of wider tokens": lambda t: torch.cat([t[..., :1], t, t[..., :2]], -1)[..., 1:-2],
    "every second token": lambda t: torch.stack([t, t * 7], 2).flatten(1, 2)[:, ::2],
    "cut off": lambda t: torch.cat([t, t], 1)[:, :t.shape[1]],
}


@pytest.mark.parametrize("view", VIEWS)
@pytest.mark.parametrize("size", [(3, 4, 33), (3, 30, 16), (2, 300, 24)], ids=str)
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_strides(gpu, size, view, dtype):
    check(gpu, *size, dtype, view=VIEWS[view])


def test_broadcast_gates_and_inputs(gpu):
    """Gates expanded over the batch: one token's distance is 0."""
    g = torch.Generator().manual_seed(3)
    x, gate = torch.randn(4, 50, 16, generator=g).cuda(), torch.randn(16, generator=g).cuda().requires_grad_()
    h, _ = gpu.gated_scan(x, gate)
    wide, _ = gpu.gated_scan(x, gate.expand(4, 50, 16))
    # the groups of tokens that are joined may be others: each is off by 16 half steps of the largest magnitude for each of up to 50 tokens
    assert (h - wide).abs().max() <= 2 * 50 * 16 * O.STEP * x.abs().max()
    w = torch.randn(4, 50, 16, generator=g).cuda()
    a, = torch.autograd.grad((h * w).sum(), gate)
    b, = torch.autograd.grad((wide * w).sum(), gate)
    # 200 terms summed in two orders
    assert (a - b).abs().max() <= 400 * O.STEP * b.abs().max() + 1e-4
    one, _ = gpu.gated_scan(x[:1].expand(4, 50, 16), gate)
    assert torch.equal(one[0], one[3]) and torch.equal(one[0], h[0])


def test_padding_is_not_looked_at(gpu):
    x, gates, s, dh, dlast = (t.cuda() for t in inputs(3, 200, 16, "f32", False, False))
    lengths = torch.tensor([0, 130, 7], device="cuda")
    leaves = [t.clone().requires_grad_() for t in (x, gates, s)]
    want = gpu.gated_scan(*leaves, lengths=lengths)
    want_grad = torch.autograd.grad(want, leaves, (dh, dlast))
    behind = torch.arange(200, device="cuda")[None, :, None] >= lengths[:, None, None]
    bad = [torch.where(behind, float("nan"), t).requires_grad_() for t in (x, gates)] + [leaves[2]]
    got = gpu.gated_scan(*bad, lengths=lengths)
    got_grad = torch.autograd.grad(got, bad, (torch.where(behind, float("inf"), dh), dlast))
    for a, b in zip(got + got_grad, want + want_grad):
        assert torch.equal(a, b)
    assert not got[0][behind.expand_as(x)].any() and torch.equal(got[1][0], s[0])


def test_sequences_do_not_meet(gpu):
    """NaN all over one sequence, also where it shares tiles with others."""
    x, gates, s, dh, dlast = (t.cuda() for t in inputs(1, 500, 16, "f32", False, False, packed=5))
    offsets = torch.tensor([0, 100, 330, 331, 460, 500], device="cuda")
    want_leaves = [t.clone().requires_grad_() for t in (x, gates, s)]
    want = gpu.gated_scan(*want_leaves, offsets=offsets)
    want_grad = torch.autograd.grad(want, want_leaves, (dh, dlast))
    for i in range(5):
        lo, hi = int(offsets[i]), int(offsets[i + 1])
        for value in (float("nan"), float("inf")):
            xb, sb = x.clone(), s.clone()
            xb[lo:hi], sb[i] = value, value
            leaves = [t.requires_grad_() for t in (xb, gates.clone(), sb)]
            got = gpu.gated_scan(*leaves, offsets=offsets)
            got_grad = torch.autograd.grad(got, leaves, (dh, dlast))
            rows, others = [t for t in range(500) if not lo <= t < hi], [j for j in range(5) if j != i]
            for a, b in zip((got[0], got_grad[0], got_grad[1]), (want[0], want_grad[0], want_grad[1])):
                assert torch.equal(a[rows], b[rows])
            assert torch.equal(got[1][others], want[1][others]) and torch.equal(got_grad[2][others], want_grad[2][others])
            assert not torch.isfinite(got[0][lo:hi]).any()


def test_what_is_not_finite_stays(gpu):
    """An infinity deep in a long sequence whose gates forget within a token: nothing behind it is finite, all before it is."""
    x, gates = torch.ones(2, 900, 8, device="cuda"), torch.full((2, 900, 8), -30.0, device="cuda")
    x[0, 37], x[1, 450] = float("inf"), float("nan")
    h, last = gpu.gated_scan(x, gates)
    for row, at in ((0, 37), (1, 450)):
        assert torch.isfinite(h[row, :at]).all() and not torch.isfinite(h[row, at:]).any() and not torch.isfinite(last[row]).any()


def test_extreme_gates(gpu):
    """+inf keeps the state, -inf takes the input, bits and all; finite ones of any size are in bounds."""
    x, s = torch.randn(1, 300, 8, device="cuda"), torch.randn(1, 8, device="cuda")
    h, last = gpu.gated_scan(x, torch.full_like(x, float("inf")), s)
    assert torch.equal(h, s[:, None].expand_as(x)) and torch.equal(last, s)
    h, last = gpu.gated_scan(x, torch.full_like(x, float("-inf")), s)
    assert torch.equal(h, x) and torch.equal(last, x[:, -1])
    gates = torch.tensor([1e30, -1e30, 87.0, -87.0, 104.0, -104.0, 0.0, -0.0], device="cuda").expand_as(x).contiguous()
    h, _ = gpu.gated_scan(x, gates, s)
    want, _, _, err, _ = O.gated_scan(x.double().cpu().numpy(), np.clip(gates.double().cpu().numpy(), -700, 700), s.double().cpu().numpy(), [(0, 0, 300)], False)
    near(h, want, err, "f32", "h")
    gates = torch.full_like(x, float("nan"))
    assert torch.isnan(gpu.gated_scan(x, gates, s)[0]).all()


@pytest.mark.parametrize("decay", [False, True])
def test_gradient_against_differences(gpu, decay):
    """Differences of the definition in 64 bits along a direction, by each input."""
    rows, length, dim = 2, 150, 9
    x, gates, s, dh, dlast = inputs(rows, length, dim, "f32", decay, False, seed=4)
    leaves = [t.cuda().requires_grad_() for t in (x, gates, s)]
    got = torch.autograd.grad(gpu.gated_scan(*leaves, decay=decay), leaves, (dh.cuda(), dlast.cuda()))
    seqs, base = O.sequences_of(rows, length), [t.double().numpy() for t in (x, gates, s)]

    def loss(values):
        h, last, _, _, _ = O.gated_scan(*values, seqs, decay)
        return (h * dh.double().numpy()).sum() + (last * dlast.double().numpy()).sum()

    errors = O.gated_scan_grad(*base, seqs, decay, dh.double().numpy(), dlast.double().numpy())[3:]
    rng = np.random.default_rng(0)
    for i in range(3):
        d = rng.standard_normal(base[i].shape)
        step = 1e-4
        up, down = [list(base), list(base)]
        up[i], down[i] = base[i] + step * d, base[i] - step * d
        want = (loss(up) - loss(down)) / (2 * step)
        mine = (got[i].double().cpu().numpy() * d).sum()
        # the difference is off by step^2 times the third derivative (by the gates up to some hundred times the first), the gradient as
        # far as its elements may be, and rounded
        size = np.abs(got[i].double().cpu().numpy() * d).sum()
        assert abs(mine - want) <= O.STEP * ((errors[i] * np.abs(d)).sum() + size) + 1e-5 * size, (i, mine, want)


@pytest.mark.parametrize("missing", ["h", "last"])
def test_one_output_used(gpu, missing):
    x, gates, s, dh, dlast = (t.cuda() for t in inputs(2, 200, 16, "f32", False, False))
    leaves = [t.requires_grad_() for t in (x, gates, s)]
    h, last = gpu.gated_scan(*leaves)
    zero = torch.zeros_like(dh), torch.zeros_like(dlast)
    want = torch.autograd.grad((h, last), leaves, (zero[0], dlast) if missing == "h" else (dh, zero[1]), retain_graph=True)
    got = torch.autograd.grad(last if missing == "h" else h, leaves, dlast if missing == "h" else dh)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("wanted", range(3))
def test_one_gradient_asked_for(gpu, wanted):
    values = [t.cuda() for t in inputs(2, 200, 16, "bf16", False, False)]
    dh, dlast = values[3:]
    leaves = [t.clone().requires_grad_() for t in values[:3]]
    want = torch.autograd.grad(gpu.gated_scan(*leaves), leaves, (dh, dlast))[wanted]
    only = [t.clone().requires_grad_(i == wanted) for i, t in enumerate(values[:3])]
    got, = torch.autograd.grad(gpu.gated_scan(*only), [only[wanted]], (dh, dlast))
    assert torch.equal(got, want)


@pytest.mark.parametrize("size", [(3, 1, 33), (3, 7, 64), (2, 40, 12), (2, 500, 20)], ids=str)
@pytest.mark.parametrize("with_lengths", [False, True])
def test_state_in_place(gpu, size, with_lengths):
    x, gates, s, _, _ = (t.cuda() for t in inputs(*size, "bf16", False, False))
    lengths = torch.tensor([0, size[1], 1][:size[0]], device="cuda") if with_lengths else None
    h, last = gpu.gated_scan(x, gates, s, lengths=lengths)
    kept = s.clone()
    version = kept._version
    h2, last2 = gpu.gated_scan(x, gates, kept, lengths=lengths, last=kept)
    assert last2 is kept and kept._version > version and torch.equal(kept, last) and torch.equal(h2, h)


MANY = [(140, 1, 1023), (140, 5, 1023), (130, 20, 1023), (260, 17, 1023), (400, 33, 1023)]      # by channels and by pieces of them, whose last two overlap


@pytest.mark.parametrize("size", MANY, ids=str)
@pytest.mark.parametrize("dtype, decay, view", [("f32", False, "time first"), ("f16", True, "part of wider tokens"), ("bf16", False, "every second token")])
def test_many_channels(gpu, size, dtype, decay, view):
    lengths = [(7 * i) % (size[1] + 1) for i in range(size[0])]
    check(gpu, *size, dtype, decay, view=VIEWS[view], lengths=lengths if decay else None, grad=size[0] == 400 and not decay)


WIDE = [("bf16", False, (64, 300, 8192)), ("f32", False, (32, 70, 8192)), ("f32", True, (260, 260, 1021)), ("f16", False, (300, 129, 1771)), ("f32", False, (16384, 130, 16)), ("bf16", True, (66000, 40, 5))]


@pytest.mark.parametrize("dtype, shared, size", WIDE, ids=str)
@pytest.mark.parametrize("with_lengths", [False, True])
def test_many_long_rows(gpu, dtype, shared, size, with_lengths):
    """Rows that one thread takes from first to last, with the states that the gradient asks for, against the same rows in parts that tiles take."""
    rows, length, dim = size
    g = torch.Generator(device="cuda").manual_seed(length)
    draw = lambda *shape: torch.randn(*shape, generator=g, device="cuda")       # noqa: E731
    x, gates, s = draw(*size).to(TYPES[dtype]), (1.0 + 3.0 * draw(dim) if shared else 1.0 + 3.0 * draw(*size)).to(TYPES[dtype]), draw(rows, dim)
    dh, dlast = draw(*size).to(TYPES[dtype]), draw(rows, dim)
    lengths = torch.arange(rows, device="cuda") * 37 % (length + 1) if with_lengths else None

    def run(rows):
        leaves = [t.detach().requires_grad_() for t in (x[rows], gates if shared else gates[rows], s[rows])]
        out = gpu.gated_scan(*leaves, lengths=lengths[rows] if with_lengths else None)
        return list(out) + list(torch.autograd.grad(out, leaves, (dh[rows], dlast[rows])))

    whole = run(slice(0, rows))
    with torch.no_grad():
        assert torch.equal(gpu.gated_scan(x, gates, s, lengths=lengths)[0], whole[0])
    for part in (slice(0, 3), slice(rows - 3, rows)):
        for i, (a, b) in enumerate(zip(whole, run(part))):
            if i == 3 and shared:
                continue
            # (tiles join their maps: other roundings, of up to 64 half steps of the largest, and one to the type)
            steps = 64 * O.STEP + (0 if a.dtype == torch.float32 else torch.finfo(a.dtype).eps)
            assert (a[part].float() - b.float()).abs().max() <= steps * b.float().abs().max().clamp(min=1), i


@pytest.mark.parametrize("size", MANY, ids=str)
def test_many_states_in_place(gpu, size):
    x, gates, s, _, _ = (t.cuda() for t in inputs(*size, "bf16", False, False))
    lengths = torch.arange(size[0], device="cuda") % (size[1] + 1)
    h, last = gpu.gated_scan(x, gates, s, lengths=lengths)
    kept = s.clone()
    h2, _ = gpu.gated_scan(x, gates, kept, lengths=lengths, last=kept)
    assert torch.equal(kept, last) and torch.equal(h2, h)


def test_steps_are_the_sequence(gpu):
    """A server's steps, one by one, some drafts at a time, and the prompt in one call: the same within roundings."""
    x, gates, s, _, _ = (t.cuda() for t in inputs(4, 60, 40, "f32", False, False))
    whole, last = gpu.gated_scan(x, gates, s)
    for each in (1, 5, 20):
        state = s.clone()
        parts = [gpu.gated_scan(x[:, t:t + each], gates[:, t:t + each], state, last=state)[0] for t in range(0, 60, each)]
        # 60 tokens of up to 16 half steps each, of magnitudes up to 4
        assert (torch.cat(parts, 1) - whole).abs().max() < 60 * 16 * 4 * O.STEP and (state - last).abs().max() < 60 * 16 * 4 * O.STEP


def test_rolled_back_to_what_was_accepted(gpu):
    """Lengths from the device: the state behind the tokens that stand, from the one before the drafts."""
    x, gates, s, _, _ = (t.cuda() for t in inputs(4, 6, 40, "bf16", False, False))
    accepted = torch.tensor([0, 3, 5, 2], dtype=torch.int32, device="cuda")
    state = s.clone()
    gpu.gated_scan(x, gates, state, lengths=accepted + 1, last=state)
    for b in range(4):
        n = int(accepted[b]) + 1
        _, want = gpu.gated_scan(x[b:b + 1, :n], gates[b:b + 1, :n], s[b:b + 1])
        assert torch.equal(state[b:b + 1], want)


def test_same_bits_every_time(gpu):
    """Tiles join as they come; the bits do not say how."""
    x, gates, s, dh, dlast = (t.cuda() for t in inputs(2, 9000, 64, "bf16", False, False))
    leaves = [t.requires_grad_() for t in (x, gates, s)]
    first = None
    for _ in range(20):
        out = gpu.gated_scan(*leaves)
        got = out + torch.autograd.grad(out, leaves, (dh, dlast))
        first = first or got
        assert all(torch.equal(a, b) for a, b in zip(got, first))


LONG = [("bf16", False, False, 33_000, 40), ("f16", False, True, 66_100, 72), ("f32", True, False, 33_100, 32), ("f32", False, True, 65_700, 20), ("bf16", True, True, 65_600, 5)]


@pytest.mark.parametrize("dtype, decay, shared, length, dim", LONG)
def test_a_long_sequence_alone_and_among_others(gpu, dtype, decay, shared, length, dim):
    """Equal bits, whether its tiles wait for one another or not, to the end of the row or not; and as several, one behind the other."""
    x, gates, s, dh, dlast = (t.cuda() for t in inputs(1, length, dim, dtype, decay, shared, seed=5))

    def run(x, gates, s, dh, dlast, **kw):
        leaves = [t.detach().requires_grad_() for t in (x, gates, s)]
        out = gpu.gated_scan(*leaves, decay=decay, **kw)
        return list(out) + list(torch.autograd.grad(out, leaves, (dh, dlast)))

    others = [t if t.dim() < 2 else torch.cat([t] + [0.5 * t] * 5) for t in (x, gates, s, dh, dlast)]
    for lengths in (None, [length], [length - 5000], [129], [0]):
        few = run(x, gates, s, dh, dlast, lengths=None if lengths is None else torch.tensor(lengths, device="cuda"))
        many = run(*others, lengths=None if lengths is None else torch.tensor(lengths * 6, device="cuda"))
        for i, (a, b) in enumerate(zip(few, many)):
            assert i == 3 and shared or torch.equal(a, b[:1]), i
    # short ones, a long one, one without tokens, tokens of none
    cuts = [7, 100, 100, 128, 5000, length - 300, length - 256, length - 3]
    n = len(cuts) - 1
    states, dstates = torch.randn(n, dim, device="cuda"), torch.randn(n, dim, device="cuda")
    flat = lambda t: t if t.dim() < 2 else t[0]                     # noqa: E731
    got = run(flat(x), flat(gates), states, flat(dh), dstates, offsets=torch.tensor(cuts, device="cuda"))
    covered = torch.zeros(length, 1, dtype=torch.bool, device="cuda")
    for i, (lo, hi) in enumerate(zip(cuts[:-1], cuts[1:])):
        cut = lambda t: t if t.dim() < 2 else t[:, lo:hi]           # noqa: E731
        one = run(cut(x), cut(gates), states[i:i + 1], cut(dh).contiguous(), dstates[i:i + 1])
        covered[lo:hi] = True
        # (tiles begin elsewhere: other roundings, of up to 64 half steps of the largest, and one to the type)
        for mine, want in ((got[0][lo:hi], one[0][0]), (got[1][i], one[1][0]), (got[2][lo:hi], one[2][0]), (got[4][i], one[4][0])):
            if want.numel():
                steps = 64 * O.STEP + (0 if want.dtype == torch.float32 else torch.finfo(want.dtype).eps)
                assert (mine.float() - want.float()).abs().max() <= steps * want.float().abs().max().clamp(min=1), i
    assert not got[0].float()[~covered.expand(-1, dim)].any() and not got[2].float()[~covered.expand(-1, dim)].any()


def test_a_long_sequence_recorded(gpu):
    x, gates, s, _, _ = (t.cuda() for t in inputs(1, 33_000, 40, "bf16", False, False, seed=6))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        gpu.gated_scan(x, gates, s)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        h, last = gpu.gated_scan(x, gates, s, last=s)
    for turn in range(4):
        x.mul_(0.5).add_(turn)
        s.fill_(float(turn))
        want, state = gpu.gated_scan(x, gates, s)
        graph.replay()
        assert torch.equal(h, want) and torch.equal(last, state) and last.data_ptr() == s.data_ptr()


def test_shapes_without_tokens(gpu):
    s = torch.randn(3, 8, device="cuda")
    h, last = gpu.gated_scan(torch.zeros(3, 0, 8, device="cuda"), torch.zeros(3, 0, 8, device="cuda"), s)
    assert h.shape == (3, 0, 8) and torch.equal(last, s) and last.data_ptr() != s.data_ptr()
    h, last = gpu.gated_scan(torch.zeros(0, 4, 8, device="cuda"), torch.zeros(8, device="cuda"))
    assert h.shape == (0, 4, 8) and last.shape == (0, 8)
    h, last = gpu.gated_scan(torch.zeros(0, 8, device="cuda"), torch.zeros(8, device="cuda"), s[:2], offsets=torch.zeros(3, dtype=torch.int32, device="cuda"))
    assert h.shape == (0, 8) and torch.equal(last, s[:2])
    gates, state = torch.zeros(8, device="cuda", requires_grad=True), s.clone().requires_grad_()
    h, last = gpu.gated_scan(torch.zeros(3, 0, 8, device="cuda"), gates, state)
    by = torch.autograd.grad(last, (gates, state), s, allow_unused=True)
    assert not by[0].any() and torch.equal(by[1], s)


def test_recorded_and_replayed(gpu):
    """Long enough for tiles that wait for one another; two graphs, other inputs at every replay, eager calls in between."""
    x, gates, s, dh, dlast = (t.cuda() for t in inputs(2, 1500, 32, "f32", False, False))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    leaves = [t.requires_grad_() for t in (x, gates, s)]

    def step():
        out = gpu.gated_scan(*leaves)
        return out + torch.autograd.grad(out, leaves, (dh, dlast))

    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graphs, outs = [], []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, pool=graphs[0].pool() if graphs else None):
            outs.append(step())
        graphs.append(g)
    for turn in range(4):
        with torch.no_grad():
            for t in leaves + [dh, dlast]:
                t.normal_()
        want = step()
        for g, out in zip(graphs, outs):
            g.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(out, want)), turn


def test_two_streams_at_once(gpu):
    args = [[t.cuda() for t in inputs(2, 3000, 64, "bf16", False, False, seed=i)][:3] for i in range(2)]
    want = [gpu.gated_scan(*a) for a in args]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in range(2)], [[], []]
    for _ in range(5):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i].append(gpu.gated_scan(*args[i]))
    torch.cuda.synchronize()
    for i in range(2):
        for out in got[i]:
            assert torch.equal(out[0], want[i][0]) and torch.equal(out[1], want[i][1])


def test_offsets_beyond_31_bits(gpu):
    """2.2 billion elements; the last sequence stands alone behind the boundary."""
    tokens, dim = 1_100_000, 2048
    g = torch.Generator(device="cuda").manual_seed(1)
    x = torch.empty(tokens, dim, device="cuda", dtype=torch.bfloat16).normal_(generator=g)
    gates = torch.empty_like(x).normal_(2.0, 1.0, generator=g)
    offsets = torch.tensor([0, tokens - 300, tokens], device="cuda")
    h, last = gpu.gated_scan(x, gates, offsets=offsets)
    tail, tail_last = gpu.gated_scan(x[None, -300:], gates[None, -300:])
    # other tiles, other joins: 300 tokens of up to 16 half steps of 32 bits, and a rounding to bf16 that may fall either way
    assert ((h[-300:].float() - tail[0].float()).abs() <= 2.0 ** -8 * tail[0].float().abs() + 300 * 16 * 4 * O.STEP).all()
    assert (last[1] - tail_last[0]).abs().max() <= 300 * 16 * 4 * O.STEP
    assert torch.equal(h[:300], gpu.gated_scan(x[:384], gates[:384])[0][:300])


def test_last_states_that_overlap_the_first(gpu):
    pool, x = torch.ones(5, 8, device="cuda"), torch.zeros(3, 40, 8, device="cuda")
    with pytest.raises(ValueError, match="last"):
        gpu.gated_scan(x, x.clone(), pool[:3], last=pool[1:4])
    h, last = gpu.gated_scan(x, x.clone(), pool[:3], last=pool[:3])              # in its place, by another view of it
    assert (last == 2.0 ** -40).all() and torch.equal(pool[:3], last) and (pool[3:] == 1).all() and (h[:, 0] == 0.5).all()
    gpu.gated_scan(x[:2], x[:2].clone(), pool[3:], last=pool[:2])


def test_refusals(gpu):
    z = lambda *shape, dtype=torch.float32: torch.zeros(*shape, device="cuda", dtype=dtype)          # noqa: E731
    x, g, s = z(2, 5, 8), z(2, 5, 8), z(2, 8)
    for bad, error in [
        (lambda: gpu.gated_scan(x, z(2, 5, 8, dtype=torch.float16)), TypeError), (lambda: gpu.gated_scan(x.double(), g.double()), TypeError),
        (lambda: gpu.gated_scan(x, z(2, 4, 8)), ValueError), (lambda: gpu.gated_scan(x, z(7)), ValueError), (lambda: gpu.gated_scan(x, z(2, 8)), ValueError),
        (lambda: gpu.gated_scan(z(8), z(8)), ValueError), (lambda: gpu.gated_scan(z(2, 5, 0), z(2, 5, 0)), ValueError),
        (lambda: gpu.gated_scan(x, g, z(3, 8)), ValueError), (lambda: gpu.gated_scan(x, g, s.half()), TypeError), (lambda: gpu.gated_scan(x, g, s.cpu()), TypeError),
        (lambda: gpu.gated_scan(x, g, lengths=z(3).int()), ValueError), (lambda: gpu.gated_scan(x, g, lengths=z(2)), TypeError),
        (lambda: gpu.gated_scan(x, g, offsets=z(3).int()), ValueError), (lambda: gpu.gated_scan(x[0], g[0], lengths=z(1).int()), ValueError),
        (lambda: gpu.gated_scan(x[0], g[0], offsets=z(1).int()), ValueError), (lambda: gpu.gated_scan(x[0], g[0], s, offsets=z(2).int()), ValueError),
        (lambda: gpu.gated_scan(x.transpose(1, 2), g.transpose(1, 2)), ValueError), (lambda: gpu.gated_scan(x, g, s, last=z(3, 8)), ValueError),
        (lambda: gpu.gated_scan(x, g, s, last=z(8, 2).t()), ValueError), (lambda: gpu.gated_scan(x.requires_grad_(), g, s, last=s), ValueError),
        (lambda: gpu.gated_scan(x.detach(), g, s, last=x.view(-1)[:16].view(2, 8)), ValueError),
    ]:
        with pytest.raises(error):
            bad()
    y = z(2, 5, 8).requires_grad_()
    h, _ = gpu.gated_scan(y, g)
    w, = torch.autograd.grad(h.sum(), y, retain_graph=True)
    with pytest.raises(RuntimeError, match="once only"):
        torch.autograd.grad(h, y, torch.ones_like(h).requires_grad_(), create_graph=True)
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(z(2, 5, 8), z(2, 5, 8))
        with pytest.raises(RuntimeError, match="forward mode"):
            gpu.gated_scan(dual, g)
