"""The token operators on the GPU against plain implementations in 64 bits.

Tolerances.  Sums of a softmax are formed by 256 threads or more, each over at most vocab / 256 + 32
terms one after the other, and exponents carry a relative error of 2 roundings: for the rows here (up to
263000 entries, logits within 100 of the largest, temperatures from 0.5) a sum is at most
1100 * 2^-24 + 300 * 2^-23 = 1.0e-4 off, a log probability or entropy as much, absolutely, and a
gradient's terms as much, relatively.  Rounding to the stored type adds half a unit of it.
"""
import numpy as np
import pytest
import torch

import token_oracles as O

pytestmark = pytest.mark.gpu

SUM = 1.0e-4
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
HALF_UNIT = {k: torch.finfo(t).eps / 2 for k, t in TYPES.items()}
LEAST = {"f32": 0.0, "bf16": 0.0, "f16": 2.0 ** -25}         # half the smallest step


def f64(t):
    return t.detach().double().cpu().numpy()


def near(got, want, size, dtype, extra=SUM):
    got = f64(got)
    bad = np.isnan(want)
    assert np.array_equal(np.isnan(got), bad)
    far = np.abs(got - want) - HALF_UNIT[dtype] * np.abs(want) * 1.01 - LEAST[dtype] - extra * size
    assert (far[~bad] <= 0).all(), "off by %g beyond the tolerance" % far[~bad].max()


def near_abs(got, want, tol):
    got = f64(got)
    assert got.shape == want.shape
    with np.errstate(over="ignore"):
        want = want.astype(np.float32).astype(np.float64)       # beyond float32's range is infinite
    bad = ~np.isfinite(want)
    assert np.array_equal(got[bad], want[bad], equal_nan=True), (got[bad][:5], want[bad][:5])
    assert np.isfinite(got[~bad]).all()
    got, want = got[~bad], want[~bad]
    assert (np.abs(got - want) <= tol * (1 + 1e-3 * np.abs(want))).all(), np.abs(got - want).max()


def gen(seed):
    return np.random.default_rng(seed)


def on_gpu(a, dtype):
    return torch.from_numpy(np.asarray(a)).to(dtype).cuda()


# ---- embedding lookup --------------------------------------------------------------------
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("n,v,d", [(1, 1, 1), (3, 5, 7), (33, 100, 64), (1000, 300, 100), (17, 40, 1023), (5, 9, 5000), (4097, 11, 8)])
def test_lookup(gpu, dtype, n, v, d):
    r = gen(n + v + d)
    table = on_gpu(r.normal(size=(v, d)), TYPES[dtype])
    ids = r.integers(-1, v, n)
    for kind in (torch.int32, torch.int64):
        got = gpu.embed(table, on_gpu(ids, kind), 1.7)
        want = torch.where(on_gpu(ids >= 0, torch.bool)[:, None], table[on_gpu(ids.clip(0), torch.int64)].float() * torch.tensor(1.7).cuda(), 0.0)
        assert got.dtype == table.dtype and torch.equal(got, want.to(table.dtype))
        near(got, O.embed(f64(table), ids, 1.7), np.abs(f64(want)), dtype, 2.0 ** -22)


def test_lookup_of_what_is_not_there(gpu):
    table = torch.randn(4, 6, device="cuda")
    ids = torch.tensor([[3, 4, -1], [2 ** 31 + 5, -2 ** 40, 0]], device="cuda")
    got = gpu.embed(table, ids, 2.0)
    assert got.shape == (2, 3, 6)
    assert torch.isnan(got[0, 1]).all() and torch.isnan(got[1, 0]).all()
    assert (got[0, 2] == 0).all() and (got[1, 1] == 0).all()
    assert torch.equal(got[0, 0], table[3] * 2) and torch.equal(got[1, 2], table[0] * 2)
    assert gpu.embed(table, ids[:, :0], 2.0).shape == (2, 0, 6)
    assert gpu.embed(table, torch.tensor(2, device="cuda")).shape == (6,)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_lookup_of_strided_rows(gpu, dtype):
    big = torch.randn(50, 77, device="cuda").to(TYPES[dtype])
    ids = torch.randint(0, 50, (2, 40), device="cuda")
    table = big[:, 3:36]                      # starts on no boundary
    assert torch.equal(gpu.embed(table, ids[1], 1.0), table[ids[1]])
    assert torch.equal(gpu.embed(table, ids.t(), 1.0), table[ids.t()])      # ids of any strides


def test_lookup_beyond_32_bits(gpu):
    table = torch.empty(1_100_000, 2048, dtype=torch.bfloat16, device="cuda")     # 2.25e9 elements
    ids = torch.tensor([0, 1_048_576, 1_099_999], device="cuda")
    table[ids] = torch.randn(3, 2048, device="cuda").bfloat16()
    assert torch.equal(gpu.embed(table, ids, 1.0), table[ids])
    grad = torch.randn(3, 2048, device="cuda").bfloat16()
    got = gpu.embed_grad(grad, ids, 1_100_000)
    assert torch.equal(got[ids], grad) and got[1:1000].count_nonzero() == 0 and got[-1000:-1].count_nonzero() == 0


# ---- its gradient ------------------------------------------------------------------------
def _grad_case(gpu, dtype, grad, ids, v, scale, out=None):
    d_grad, d_ids = on_gpu(grad, TYPES[dtype]), on_gpu(ids, torch.int64)
    want, size, count = O.embed_grad(f64(d_grad), ids, v, scale)
    got = gpu.embed_grad(d_grad, d_ids, v, scale)
    # a row's sum is off by a rounding for each of its tokens at most, and one for the factor
    near(got, want, size, dtype, (count[:, None] + 2) * 2.0 ** -24)
    assert torch.equal(got, gpu.embed_grad(d_grad, d_ids.int(), v, scale))      # the same bits again
    base = torch.randn(v, grad.shape[1], device="cuda")
    into = base.clone()
    assert gpu.embed_grad(d_grad, d_ids, v, scale, out=into) is into
    near(into, want + f64(base), size + np.abs(f64(base)), "f32", (count[:, None] + 2) * 2.0 ** -24)
    assert torch.equal(into[on_gpu(count == 0, torch.bool)], base[on_gpu(count == 0, torch.bool)])


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("n,v,d", [(1, 1, 1), (2, 3, 5), (31, 4, 64), (33, 1, 100), (65, 2, 9), (1000, 300, 100), (2049, 5000, 33),
                                   (3000, 7, 513), (700, 2500, 1025)])
def test_lookup_gradient(gpu, dtype, n, v, d):
    r = gen(n * v + d)
    _grad_case(gpu, dtype, r.normal(size=(n, d)), r.integers(-1, v + 1, n), v, 0.37)


@pytest.mark.parametrize("counts", [[32], [33], [31, 33], [64, 65, 1], [1, 32, 200, 1, 96, 500, 2], [1025] * 3, [0, 0, 40, 0]])
def test_lookup_gradient_of_common_tokens(gpu, counts):
    """Rows with as many tokens as a piece holds, one more, several pieces, in and out of order."""
    r = gen(sum(counts))
    ids = np.repeat(np.arange(len(counts)), counts)
    _grad_case(gpu, "f32", r.normal(size=(len(ids), 70)), ids, len(counts), 1.0)
    _grad_case(gpu, "bf16", r.normal(size=(len(ids), 70)), r.permutation(ids), len(counts), 1.0)


def test_lookup_gradient_without_tokens(gpu):
    grad = torch.full((5, 12), float("nan"), device="cuda")
    none = torch.full((5,), -1, device="cuda")
    assert torch.equal(gpu.embed_grad(grad, none, 9), torch.zeros(9, 12, device="cuda"))
    assert torch.equal(gpu.embed_grad(grad[:0], none[:0], 9), torch.zeros(9, 12, device="cuda"))
    out = torch.randn(9, 12, device="cuda")
    assert torch.equal(gpu.embed_grad(grad, none, 9, out=out.clone()), out)


def test_lookup_gradient_by_autograd(gpu):
    table = torch.randn(30, 16, device="cuda", requires_grad=True)
    ids = torch.randint(0, 30, (4, 25), device="cuda")
    gpu.embed(table, ids, 0.5).sum().backward()          # a broadcast gradient
    count = torch.bincount(ids.flatten(), minlength=30).float()
    assert torch.allclose(table.grad, (0.5 * count)[:, None].expand(-1, 16), rtol=1e-6)
    strided = torch.randn(100, 2, 16, device="cuda")[:, 1]
    want, _, _ = O.embed_grad(f64(strided), ids.flatten().cpu().numpy(), 30, 1.0)
    near(gpu.embed_grad(strided, ids.flatten(), 30), want, np.abs(want) + 10, "f32", 1e-6)
    x = gpu.embed(table, ids)
    g, = torch.autograd.grad(x, table, torch.ones_like(x).requires_grad_(), create_graph=False)
    with pytest.raises(RuntimeError, match="once"):
        torch.autograd.grad(gpu.embed(table, ids), table, torch.ones_like(x).requires_grad_(), create_graph=True)


@pytest.mark.parametrize("n,v,d,dtype", [(2048, 5, 40, "bf16"), (2049, 5, 40, "bf16"), (4097, 300_000, 24, "f32"), (70_000, 20_000, 40, "f16"),
                                         (5000, 2_200_000, 4, "f32"), (200_000, 3, 8, "f32"), (9000, 70, 1030, "f16"), (2500, 3_000_000, 3, "bf16")])
def test_lookup_gradient_of_many_tokens(gpu, n, v, d, dtype):
    """Tokens in chunks and buckets, more rows than a bucket counts at a time, every seventh token of one row."""
    r = gen(n)
    ids = np.where(np.arange(n) % 7 == 3, v // 2, r.integers(-1, v + 1, n))
    d_ids, grad = on_gpu(ids, torch.int64), on_gpu(r.normal(size=(n, d)).astype(np.float32), TYPES[dtype])
    got = gpu.embed_grad(grad, d_ids, v, 0.5)
    valid = (d_ids >= 0) & (d_ids < v)
    want = torch.zeros(v, d, dtype=torch.float64, device="cuda").index_add_(0, d_ids[valid], grad[valid].double() * 0.5)
    size = torch.zeros(v, d, dtype=torch.float64, device="cuda").index_add_(0, d_ids[valid], grad[valid].double().abs() * 0.5)
    count = torch.bincount(d_ids[valid], minlength=v).double()[:, None]
    far = (got.double() - want).abs() - HALF_UNIT[dtype] * want.abs() * 1.01 - LEAST[dtype] - (count + 2) * 2.0 ** -24 * size
    assert (far <= 0).all() and torch.equal(got, gpu.embed_grad(grad, d_ids.int(), v, 0.5))
    base = torch.randn(v, d, device="cuda")
    into = gpu.embed_grad(grad, d_ids, v, 0.5, out=base.clone())
    far = (into.double() - want - base.double()).abs() - ((count + 3) * 2.0 ** -24) * (size + base.double().abs())
    assert (far <= 0).all() and torch.equal(into[count[:, 0] == 0], base[count[:, 0] == 0])


def test_many_tokens_of_few_rows(gpu):
    n, d = 131_072, 24
    ids = torch.zeros(n, dtype=torch.int64, device="cuda")
    ids[::3] = 1
    grad = torch.randn(n, d, device="cuda")
    got = gpu.embed_grad(grad, ids, 3)
    want = torch.stack([grad[ids == 0].double().sum(0), grad[ids == 1].double().sum(0), torch.zeros(d, device="cuda").double()])
    # sums of 32, then of those: no chain is longer than 32 + 4096 / 4 + 4
    assert ((got.double() - want).abs() <= 1100 * 2.0 ** -24 * n).all()
    assert ((got.double() - want).abs() <= 1e-2).all()


# ---- log probabilities -------------------------------------------------------------------
LOGIT_SHAPES = [(1, 1), (2, 2), (3, 7), (5, 64), (2, 2047), (2, 2048), (3, 2049), (1, 4097), (70, 1000), (1100, 33), (3, 20_011), (1, 70_000),
                (1, 262_145), (1030, 2500)]


def _logits(r, n, v):
    z = r.normal(size=(n, v)) * 3
    z[:, r.integers(0, v)] += 8
    if n > 2:
        z[1, r.random(v) < 0.9] = -np.inf
        z[2] = np.round(z[2])                 # many ties
    return z


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("n,v", LOGIT_SHAPES)
def test_token_logprobs(gpu, dtype, n, v):
    r = gen(n * 7 + v)
    z = on_gpu(_logits(r, n, v), TYPES[dtype])
    targets = r.integers(-1, v, n)
    for top, temperature in ((0, 1.0), (min(v, 1), 0.5), (min(v, 20), 1.3), (min(v, 64), 1.0)):
        want = O.token_logprobs(f64(z), targets, top, temperature)
        got = gpu.token_logprobs(z, on_gpu(targets, torch.int32), top, temperature)
        assert len(got) == (4 if top else 2)
        near_abs(got[0], want[0], SUM)
        near_abs(got[1], want[1], 20 * SUM)         # its terms reach log v + 1 times a probability's error
        if top:
            assert np.array_equal(got[2].cpu().numpy(), want[2])
            near_abs(got[3], want[3], SUM)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("n,v", LOGIT_SHAPES)
def test_token_logprobs_gradient(gpu, dtype, n, v):
    r = gen(n * 5 + v)
    z = on_gpu(_logits(r, n, v), TYPES[dtype]).requires_grad_()
    targets = r.integers(-1, v, n)
    g, h = r.normal(size=n), r.normal(size=n)
    if n > 4:
        g[3] = h[3] = 0
    d_g, d_h = on_gpu(g, torch.float32), on_gpu(h, torch.float32)
    lp, entropy = gpu.token_logprobs(z, on_gpu(targets, torch.int64), temperature=0.8)
    for grads, factors in (((d_g, d_h), (f64(d_g), f64(d_h))), ((d_g, None), (f64(d_g), 0 * h)), ((None, d_h), (0 * g, f64(d_h)))):
        outs = [(o, w) for o, w in zip((lp, entropy), grads) if w is not None]
        dz, = torch.autograd.grad([o for o, _ in outs], z, [w for _, w in outs], retain_graph=True)
        want, size = O.token_logprobs_grad(f64(z), targets, 0.8, *factors)
        assert dz.dtype == z.dtype
        near(dz, want, size, dtype)


def test_rows_that_say_nothing(gpu):
    inf, low = float("inf"), torch.finfo(torch.float32).min
    z = torch.randn(8, 1000, device="cuda")
    z[0] = -inf
    z[1] = low                       # the type's lowest value everywhere: all alike
    z[2, 5] = float("nan")
    z[3, 5] = inf
    z[4] = -inf
    z[4, 700] = 3.0
    z[5] = low
    z[5, 10:12] = 1.0
    z[6, ::2] = low
    z[7] = float("nan")
    z.requires_grad_()
    targets = torch.tensor([3, 3, 3, 5, 700, 10, 1, 0], device="cuda")
    lp, entropy, ids, lps = gpu.token_logprobs(z, targets, 4, 0.5)
    want = O.token_logprobs(f64(z), targets.cpu().numpy(), 4, 0.5)
    near_abs(lp, np.array([-inf, *want[0][1:]]), SUM)
    near_abs(entropy, np.array([0.0, *want[1][1:]]), 20 * SUM)
    rows = [0, 1, 4, 5, 6]
    assert np.array_equal(ids.cpu().numpy()[rows], want[2][rows])
    near_abs(lps[rows], want[3][rows], SUM)
    assert torch.isnan(lps[[2, 3, 7]]).all()
    assert torch.equal(ids[7].cpu(), torch.arange(4, dtype=torch.int32)) and 5 not in ids[2].tolist() and ids[3, 0] == 5
    dz, = torch.autograd.grad((lp, entropy), z, (torch.ones_like(lp), torch.ones_like(lp)))
    ref, size = O.token_logprobs_grad(f64(z), targets.cpu().numpy(), 0.5, np.ones(8), np.ones(8))
    near(dz, ref, size, "f32")
    assert (dz[0] == 0).all() and (dz[4] == 0).all()


def test_alternatives_in_any_order(gpu):
    """Rows that ascend, descend, hold one value only, or put the best into one thread's hands."""
    v = 9000
    z = torch.zeros(7, v, device="cuda")
    z[0] = torch.arange(v)
    z[1] = -torch.arange(v)
    z[2] = 2.0
    z[3, 4000:4064] = 1.0
    z[4, 8::2048] = 5.0
    z[5] = torch.where(torch.arange(v) % 2 == 0, 0.0, -0.0)
    z[6, -1] = -1e30
    z[6, 77] = 1e30
    targets = torch.zeros(7, dtype=torch.int64, device="cuda")
    for rows in (z, z.repeat(300, 1)):           # split over workgroups, and one workgroup a row
        for top in (1, 63, 64):
            ids = gpu.token_logprobs(rows, targets.repeat(rows.shape[0] // 7), top)[2]
            want = torch.sort(rows, dim=1, descending=True, stable=True).indices[:, :top]
            assert torch.equal(ids.long(), want)


# ---- distillation ------------------------------------------------------------------------
def _teacher(r, n, v, k, spread):
    ids = r.integers(0, max(1, min(v, spread)), (n, k))
    teacher = r.normal(size=(n, k)) * 2
    ids[r.random((n, k)) < 0.15] = -1
    teacher[r.random((n, k)) < 0.1] = -np.inf
    if n > 2:
        ids[2] = -1
        teacher[2, :] = np.nan                   # in slots that are empty
    return ids, teacher


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("n,v", LOGIT_SHAPES)
@pytest.mark.parametrize("k,spread", [(1, 10 ** 9), (10, 6), (65, 10 ** 9), (300, 40)])
def test_distillation(gpu, dtype, n, v, k, spread):
    r = gen(n * 3 + v + k)
    z = on_gpu(_logits(r, n, v), TYPES[dtype])
    if n > 2:
        z[1] = z[0]                              # no token ruled out: the losses are numbers
    ids, teacher = _teacher(r, n, v, k, spread)
    weights = r.normal(size=n)
    if n > 4:
        weights[4] = 0
    d_ids, d_teacher, d_w = on_gpu(ids, torch.int64), on_gpu(teacher, torch.float32), on_gpu(weights, torch.float32)
    want, ref, size = O.distill(f64(z), ids, f64(d_teacher), 1.5, f64(d_w))
    loss = gpu.distill_loss(z, d_ids, d_teacher, 1.5)
    near_abs(loss, want, 2 * SUM)
    assert loss.dtype == torch.float32
    losses, grad = gpu.distill_step(z, d_ids.int(), d_teacher, d_w, 1.5)
    near_abs(losses, want, 2 * SUM)
    near(grad, ref, size, dtype)
    z.requires_grad_()
    dz, = torch.autograd.grad(gpu.distill_loss(z, d_ids, d_teacher, 1.5), z, d_w)
    near(dz, ref, size, dtype)


# Rows that a workgroup holds, by every number of threads and pieces, more rows than workgroups, rows just too long.
@pytest.mark.parametrize("n,v,k,dtype", [
    (5, 8, 3, "f16"), (5, 9, 3, "bf16"), (3, 4, 2, "f32"), (40, 2047, 64, "f16"), (40, 4100, 64, "bf16"), (40, 8191, 64, "f16"), (40, 8190, 65, "bf16"),
    (40, 16_000, 100, "f16"), (40, 32_767, 256, "bf16"), (40, 16_383, 100, "f32"), (40, 20_000, 300, "f16"), (97, 50_001, 512, "f16"),
    (97, 65_533, 10, "bf16"), (40, 30_000, 600, "f16"), (97, 60_000, 1024, "bf16"), (97, 81_917, 64, "f16"), (97, 106_001, 64, "bf16"),
    (97, 131_072, 64, "bf16"), (97, 65_536, 64, "f32"), (97, 131_080, 64, "bf16"), (300, 66_001, 20, "f16"), (6200, 40, 5, "f32"), (1100, 9000, 70, "f16")])
def test_distillation_by_rows(gpu, n, v, k, dtype):
    r = gen(n + v + k)
    z = on_gpu((r.normal(size=(n, v)) * 2).astype(np.float32), TYPES[dtype])
    ids, teacher = _teacher(r, n, v, k, max(2, v // 3))
    weights = np.where(r.random(n) < 0.1, 0.0, r.normal(size=n))
    d_teacher, d_w = on_gpu(teacher, torch.float32), on_gpu(weights, torch.float32)
    want, ref, size = O.distill(f64(z), ids, f64(d_teacher), 0.7, f64(d_w))
    losses, grad = gpu.distill_step(z, on_gpu(ids, torch.int64), d_teacher, d_w, 0.7)
    near_abs(losses, want, 2 * SUM)
    near(grad, ref, size, dtype)
    assert torch.equal(gpu.distill_step(z, on_gpu(ids, torch.int32), d_teacher, d_w, 0.7, out=z)[1], grad) and torch.equal(z, grad)


# One wavefront a row: enough rows, or short ones.
@pytest.mark.parametrize("n,v,dtype", [(4100, 801, "f16"), (4096, 2049, "bf16"), (4097, 1500, "f32"), (2000, 2047, "bf16"), (1500, 1024, "f32"), (5000, 4111, "f16")])
def test_token_logprobs_by_wavefronts(gpu, n, v, dtype):
    r = gen(n + v)
    z = on_gpu(_logits(r, n, v).astype(np.float32), TYPES[dtype])
    targets = r.integers(-1, v, n)
    for top in (0, 7, 64):
        want = O.token_logprobs(f64(z), targets, top, 0.9)
        got = gpu.token_logprobs(z, on_gpu(targets, torch.int64), top, 0.9)
        near_abs(got[0], want[0], SUM)
        near_abs(got[1], want[1], 20 * SUM)
        if top:
            assert np.array_equal(got[2].cpu().numpy(), want[2])
            near_abs(got[3], want[3], SUM)


@pytest.mark.parametrize("teacher_dtype", ["f32", "bf16", "f16"])
def test_distillation_most_slots(gpu, teacher_dtype):
    r = gen(5)
    z, ids = on_gpu(r.normal(size=(3, 5000)), torch.bfloat16), r.integers(0, 5000, (3, 1024))
    teacher = on_gpu(r.normal(size=(3, 1024)), TYPES[teacher_dtype])
    want, ref, size = O.distill(f64(z), ids, f64(teacher), 1.0, np.ones(3))
    losses, grad = gpu.distill_step(z, on_gpu(ids, torch.int64), teacher)
    near_abs(losses, want, 2 * SUM)
    near(grad, ref, size, "bf16")


@pytest.mark.parametrize("n", [9, 1500])
def test_distillation_of_rows_that_say_nothing(gpu, n):
    inf, nan = float("inf"), float("nan")
    z = torch.randn(9, 700, device="cuda")
    ids = torch.randint(0, 700, (9, 5), device="cuda")
    ids[:, 0] = 3
    teacher = torch.randn(9, 5, device="cuda")
    z[0] = -inf                                  # nothing left for the student
    z[1, 3] = -inf                               # ruled out, and the teacher's
    z[2, 9] = nan
    teacher[3] = -inf                            # no teacher
    z[4] = nan
    ids[4] = -1                                  # no teacher, and no numbers
    ids[5, 2] = 700                              # beyond the vocabulary
    ids[6, 2], teacher[6, 2] = 900, -inf         # beyond it in an empty slot
    z[7] = torch.finfo(torch.float32).min
    z[7, :2] = 0.0
    ids[7] = torch.tensor([0, 1, 1, 0, 1], device="cuda")
    teacher[8, 1] = nan
    want, ref, size = O.distill(f64(z), ids.cpu().numpy(), f64(teacher), 1.0, np.ones(9))
    want[0] = inf
    z, ids, teacher = (t.repeat(-(-n // 9), 1)[:n] for t in (z, ids, teacher))
    losses, grad = gpu.distill_step(z, ids, teacher)
    z2 = z.clone().requires_grad_()
    dz, = torch.autograd.grad(gpu.distill_loss(z2, ids, teacher).sum(), z2)
    for i in range(0, n, 9):
        near_abs(losses[i:i + 9][:n - i], want[:n - i], 2 * SUM)
        near(grad[i:i + 9], ref[:n - i], size[:n - i], "f32")
        near(dz[i:i + 9], ref[:n - i], size[:n - i], "f32")
    assert torch.isinf(losses[1]) and torch.isnan(losses[5]) and torch.isfinite(losses[6])


@pytest.mark.parametrize("n,v", [(3, 5000), (2000, 1001), (300, 140_001)])
def test_gradient_in_the_logits_place(gpu, n, v):
    z = torch.randn(n, v, device="cuda").bfloat16()
    ids, teacher = torch.randint(0, v, (n, 20), device="cuda"), torch.randn(n, 20, device="cuda")
    ids[:, 10:] = ids[:, :10]
    losses, grad = gpu.distill_step(z, ids, teacher)
    again, same = gpu.distill_step(z, ids, teacher, out=z)
    assert same is z and torch.equal(again, losses) and torch.equal(z, grad)


def test_strides_and_leading_shapes(gpu):
    big = torch.randn(6, 10, 1031, device="cuda").half()
    z = big[:, :, 5:1026]                        # rows at a distance, off any boundary
    t = torch.randint(0, 1021, (10, 6), device="cuda").t()
    ids, teacher = torch.randint(0, 1021, (6, 10, 8), device="cuda"), torch.randn(8, 6, 10, device="cuda").permute(1, 2, 0)
    flat = z.reshape(60, 1021).contiguous()
    for a, b in zip(gpu.token_logprobs(z, t, 3), gpu.token_logprobs(flat, t.reshape(-1), 3)):
        assert a.shape[:2] == (6, 10) and torch.equal(a.flatten(0, 1), b)
    a = gpu.distill_step(z, ids, teacher)
    b = gpu.distill_step(flat, ids.reshape(60, 8), teacher.reshape(60, 8))
    assert torch.equal(a[0].flatten(), b[0]) and torch.equal(a[1].flatten(0, 1), b[1])
    out = torch.zeros(6, 10, 1100, device="cuda").half()
    gpu.distill_step(z, ids, teacher, out=out[:, :, 7:1028])
    assert torch.equal(out[:, :, 7:1028].flatten(0, 1), b[1]) and (out[:, :, :7] == 0).all() and (out[:, :, 1028:] == 0).all()
    one = gpu.token_logprobs(z[2, 3], t[2, 3], 3)
    assert one[0].shape == () and one[2].shape == (3,)
    none = gpu.token_logprobs(z[:0], t[:0], 3)
    assert none[0].shape == (0, 10) and none[3].shape == (0, 10, 3)
    assert gpu.distill_step(z[:0], ids[:0], teacher[:0])[1].shape == (0, 10, 1021)


def test_rows_beyond_32_bits(gpu):
    step = 2 ** 30 + 24
    store = torch.zeros(2 * step + 2000, dtype=torch.bfloat16, device="cuda")
    z = store.as_strided((3, 1500), (step, 1))
    z.copy_(torch.randn(3, 1500, device="cuda"))
    near_z = z.contiguous()
    t = torch.tensor([1, 2, 1499], device="cuda")
    ids, teacher = torch.randint(0, 1500, (3, 4), device="cuda"), torch.randn(3, 4, device="cuda")
    for a, b in zip(gpu.token_logprobs(z, t, 5), gpu.token_logprobs(near_z, t, 5)):
        assert torch.equal(a, b)
    want = gpu.distill_step(near_z, ids, teacher)
    got = gpu.distill_step(z, ids, teacher, out=z)
    assert torch.equal(got[0], want[0]) and torch.equal(z, want[1])


def test_gradients_against_differences(gpu):
    r = gen(3)
    v, e = 6, 1e-2
    z = on_gpu(r.normal(size=(1, v)), torch.float32)
    t = torch.tensor([2], device="cuda")
    ids, teacher = torch.tensor([[1, 4, 1]], device="cuda"), torch.tensor([[0.3, -0.5, 1.0]], device="cuda")

    def values(x):
        lp, entropy = gpu.token_logprobs(x, t, temperature=0.9)
        return torch.stack([lp[0], entropy[0], gpu.distill_loss(x, ids, teacher, 0.9)[0]])

    x = z.clone().requires_grad_()
    exact = torch.stack([torch.autograd.grad(values(x)[i], x)[0][0] for i in range(3)])
    for j in range(v):
        up, down = z.clone(), z.clone()
        up[0, j] += e
        down[0, j] -= e
        # third derivatives below 2, values to 1e-6
        diff = (values(up) - values(down)) / (2 * e)
        assert (diff - exact[:, j]).abs().max() < 2 * e * e + 1e-6 / e


def test_streams_and_graphs(gpu):
    z = torch.randn(40, 9001, device="cuda").bfloat16()
    t, ids, teacher = torch.randint(0, 9001, (40,), device="cuda"), torch.randint(0, 9001, (40, 12), device="cuda"), torch.randn(40, 12, device="cuda")
    table, grad = torch.randn(500, 40, device="cuda"), torch.randn(900, 40, device="cuda")
    toks = torch.randint(0, 500, (900,), device="cuda")

    def work():
        return [*gpu.token_logprobs(z, t, 7), *gpu.distill_step(z, ids, teacher), gpu.embed(table, toks, 3.0), gpu.embed_grad(grad, toks, 500)]

    want = [x.clone() for x in work()]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = work()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = work()
    for i in range(4):
        z.copy_(torch.randn(40, 9001, device="cuda").bfloat16() * (i + 1))
        toks.copy_(torch.randint(0, 500, (900,), device="cuda"))
        want = [x.clone() for x in work()]
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want)), i


def test_refusals(gpu):
    z, t = torch.randn(4, 9, device="cuda"), torch.zeros(4, dtype=torch.int64, device="cuda")
    ids, teacher = torch.zeros(4, 3, dtype=torch.int64, device="cuda"), torch.zeros(4, 3, device="cuda")
    table = torch.randn(5, 8, device="cuda")
    for call in (lambda: gpu.embed(table.double(), t), lambda: gpu.embed(table, t.float()), lambda: gpu.embed(table.cpu(), t),
                 lambda: gpu.embed(table, t.cpu()), lambda: gpu.embed_grad(z, t, 5, out=torch.zeros(5, 9, device="cuda").half()),
                 lambda: gpu.token_logprobs(z.int(), t), lambda: gpu.token_logprobs(z, t.short()),
                 lambda: gpu.distill_step(z, ids, teacher, torch.ones(4, device="cuda").double()),
                 lambda: gpu.distill_loss(z, ids, teacher.double())):
        with pytest.raises(TypeError):
            call()
    for call in (lambda: gpu.embed(table.t(), t), lambda: gpu.embed(table[0], t), lambda: gpu.embed(table[:0], t),
                 lambda: gpu.embed(table[:1].expand(5, 8), t), lambda: gpu.embed_grad(z, t[:3], 5), lambda: gpu.embed_grad(z, t, 0),
                 lambda: gpu.embed_grad(z, t, 5, out=torch.zeros(5, 8, device="cuda")), lambda: gpu.embed_grad(z, t, 4, out=z),
                 lambda: gpu.embed_grad(z, t, 5, out=torch.zeros(9, 5, device="cuda").t()),
                 lambda: gpu.token_logprobs(z, t[:3]), lambda: gpu.token_logprobs(z, t, 10), lambda: gpu.token_logprobs(z, t, -1),
                 lambda: gpu.token_logprobs(torch.randn(4, 99, device="cuda"), t, 65), lambda: gpu.token_logprobs(z, t, 0, 0.0),
                 lambda: gpu.token_logprobs(z, t, 0, float("nan")), lambda: gpu.token_logprobs(z, t, 0, -1.0),
                 lambda: gpu.token_logprobs(z.t().contiguous().t(), t), lambda: gpu.token_logprobs(z[:, :0], t),
                 lambda: gpu.token_logprobs(torch.randn(3, 2, 9, device="cuda").transpose(0, 1), torch.zeros(2, 3, dtype=torch.int64, device="cuda")),
                 lambda: gpu.distill_loss(z, ids[:, :0], teacher[:, :0]), lambda: gpu.distill_loss(z, ids, teacher[:, :2]),
                 lambda: gpu.distill_loss(z, ids[:3], teacher[:3]), lambda: gpu.distill_loss(z, ids, teacher, float("inf")),
                 lambda: gpu.distill_loss(z, ids.repeat(1, 400), teacher.repeat(1, 400)),
                 lambda: gpu.distill_loss(z, ids, teacher.clone().requires_grad_()),
                 lambda: gpu.distill_step(z, ids, teacher, torch.ones(3, device="cuda")), lambda: gpu.distill_step(z, ids, teacher, out=z[:3]),
                 lambda: gpu.distill_step(z, ids, teacher, out=z.half()),
                 lambda: gpu.distill_step(z[:2], ids[:2], teacher[:2], out=z[1:3])):
        with pytest.raises(ValueError):
            call()


# ---- where one way of computing ends and the next begins ---------------------------------
@pytest.mark.parametrize("n,v,k,dtype", [(1023, 5000, 10, "f16"), (1024, 5001, 64, "bf16"), (1100, 8191, 33, "f16"), (1024, 4095, 7, "f32")])
def test_distillation_by_wavefronts(gpu, n, v, k, dtype):
    test_distillation_by_rows(gpu, n, v, k, dtype)


@pytest.mark.parametrize("dtype,n,v", [("bf16", 3, 16_376), ("f16", 3, 16_385), ("bf16", 2, 16_392), ("f32", 2, 8192), ("f32", 2, 8193), ("f16", 600, 17_001)])
def test_token_logprobs_about_the_longest_row_of_one_workgroup(gpu, dtype, n, v):
    test_token_logprobs(gpu, dtype, n, v)


@pytest.mark.parametrize("n,v,d,dtype", [(30_000, 300_000, 20, "f32"), (30_000, 900, 72, "bf16"), (5000, 40, 9, "f16")])
def test_lookup_gradient_of_half_the_tokens_one_row(gpu, n, v, d, dtype):
    r = gen(n + d)
    ids = np.where(r.random(n) < 0.5, 7, r.integers(0, v, n))
    _grad_case(gpu, dtype, r.normal(size=(n, d)), ids, v, 1.0)
    ids[:] = 7
    ids[n // 2:n // 2 + 100] = r.integers(0, v, 100)
    _grad_case(gpu, dtype, r.normal(size=(n, d)), ids, v, 1.0)


@pytest.mark.parametrize("n,v,d", [(1, 3, 1), (300, 40, 33), (6000, 500, 16)])
def test_lookup_gradient_against_differences(gpu, n, v, d):
    """The lookup is linear: with small whole numbers sum G (embed(W + E) - embed(W)) = sum E embed_grad(G), bit by bit."""
    r = gen(n)
    table, step, grad = (on_gpu(r.integers(-4, 5, shape), torch.float32) for shape in ((v, d), (v, d), (n, d)))
    ids = on_gpu(r.integers(-1, v, n), torch.int64)
    rise = (grad.double() * (gpu.embed(table + step, ids, 0.5) - gpu.embed(table, ids, 0.5)).double()).sum()
    assert rise == (step.double() * gpu.embed_grad(grad, ids, v, 0.5).double()).sum()


# Rows of one group of threads that is no power of two, of two that share them in whole lines, of parts of runs.
@pytest.mark.parametrize("n,v,d,dtype", [(40, 700, 624, "f16"), (300, 700, 625, "bf16"), (257, 9, 520, "f32"), (5000, 300, 168, "bf16"), (6000, 100, 1000, "f16"),
                                         (4100, 90, 1333, "f32"), (256, 5000, 21, "f16"), (3000, 2000, 1030, "bf16")])
def test_lookup_and_its_gradient_of_uneven_rows(gpu, n, v, d, dtype):
    r = gen(n + v + d)
    _grad_case(gpu, dtype, r.normal(size=(n, d)), r.integers(-1, v, n), v, 1.0)
    table = on_gpu(r.normal(size=(v, d)), TYPES[dtype])
    ids = on_gpu(r.integers(0, v, n), torch.int64)
    assert torch.equal(gpu.embed(table, ids), table[ids])


@pytest.mark.parametrize("n,v,d,dtype", [(4097, 40_000, 5, "f16"), (4200, 33_700, 7, "f32"), (9000, 72_000, 3, "bf16"), (9000, 71_999, 3, "bf16")])
def test_lookup_gradient_by_a_table_that_stays_empty(gpu, n, v, d, dtype):
    r = gen(v)
    _grad_case(gpu, dtype, r.normal(size=(n, d)), r.integers(-1, v + 1, n), v, 2.0)
    got = gpu.embed_grad(torch.zeros(n, d, device="cuda", dtype=TYPES[dtype]), torch.full((n,), -1, device="cuda"), v)
    assert not got.any()


def test_lookup_gradient_of_few_tokens_by_a_large_table(gpu):
    """One that a launch of its own clears: zeros everywhere but in the tokens' rows, to the last element."""
    v, d = 800_001, 253                    # 810 MB
    r = gen(9)
    ids = np.concatenate([r.integers(0, v, 40), [0, v - 1, v - 1, -1, v]])
    grad = on_gpu(r.normal(size=(45, d)), torch.float32)
    got = gpu.embed_grad(grad, on_gpu(ids, torch.int64), v)
    want = torch.zeros(v, d, device="cuda", dtype=torch.float64)
    real = on_gpu((ids >= 0) & (ids < v), torch.bool)
    want.index_add_(0, on_gpu(ids, torch.int64)[real], grad[real].double())
    assert ((got.double() - want).abs() <= 2 * 2.0 ** -23 * want.abs().clamp(max=8)).all()
    del want
    assert torch.equal(gpu.embed_grad(grad, on_gpu(ids, torch.int64), v, out=torch.zeros_like(got)), got)


# Every number of threads, more rows than workgroups: wavefronts hand over sums, losses and slots of one row after the other.
@pytest.mark.parametrize("n,v,k,dtype", [(7000, 1500, 64, "f16"), (3000, 4001, 200, "bf16"), (2000, 30_001, 130, "f16"), (1200, 60_000, 300, "bf16"), (700, 30_000, 900, "f32")])
def test_distillation_of_many_rows_is_the_same_again(gpu, n, v, k, dtype):
    """Losses far from the rows' sums, rows alike but for their place: a sum taken for another's would show."""
    z = (40 * torch.rand(3, v, device="cuda")).to(TYPES[dtype]).repeat(-(-n // 3), 1)[:n]
    ids, teacher = (t.repeat(-(-n // 3), 1)[:n] for t in (torch.randint(0, v, (3, k), device="cuda"), torch.randn(3, k, device="cuda")))
    first = gpu.distill_step(z, ids, teacher)
    for i in range(3):
        losses, grad = gpu.distill_step(z, ids, teacher)
        assert torch.equal(losses, first[0]) and torch.equal(grad, first[1])
        assert torch.equal(losses, losses[:3].repeat(-(-n // 3))[:n]) and torch.equal(grad, grad[:3].repeat(-(-n // 3), 1)[:n])


# Logits at the lowest value of their type: what the definition gives is a number wherever float32 holds it, and is returned.
# (Off by the rounding of the difference, of the quotient and of the stored value: 2^-22 of it, beside what a sum is off.)
def _all_near(got, want):
    got = f64(got)
    with np.errstate(over="ignore"):
        beyond = np.isinf(want.astype(np.float32))
    assert np.array_equal(np.isinf(got), beyond) and np.array_equal(got[beyond] > 0, want[beyond] > 0), (got, want)
    far = np.abs(got - want)[~beyond] - 2 * SUM - 2.0 ** -22 * np.abs(want[~beyond])
    assert (far <= 0).all(), far.max()


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("temperature", [0.9, 1.0, 1.2, 3.0])
@pytest.mark.parametrize("n,v", [(3, 200), (2, 33_000), (4100, 320)])
def test_log_probabilities_of_the_lowest_logits(gpu, dtype, temperature, n, v):
    r = gen(v)
    z = on_gpu(r.normal(size=(n, v)), TYPES[dtype])
    z[:, 5:] = torch.finfo(TYPES[dtype]).min
    if dtype != "f16":
        z[1, :3] = 1e38                          # a difference beyond float32; its quotient by 3 is not
    targets = r.integers(0, v, n)
    want = O.token_logprobs(f64(z), targets, 8, temperature)
    got = gpu.token_logprobs(z, on_gpu(targets, torch.int64), 8, temperature)
    assert np.array_equal(got[2].cpu().numpy(), want[2])
    for i in (0, 1, 3):
        _all_near(got[i], want[i])
    if dtype != "f16" and temperature == 1.0:
        finite = torch.isfinite(torch.log_softmax(z.float(), 1).gather(1, on_gpu(targets, torch.int64)[:, None])[:, 0])
        assert torch.isfinite(got[0][finite]).all() and finite[0]


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("temperature", [0.9, 1.0, 3.0])
@pytest.mark.parametrize("n,v", [(5, 300), (5, 9000), (5, 140_000), (100, 70_000)])
def test_distillation_to_the_lowest_logits(gpu, dtype, temperature, n, v):
    """The teacher names tokens that the student's mask has at the type's lowest value: one of them, some, all."""
    r = gen(v + n)
    z = on_gpu(r.normal(size=(n, v)), TYPES[dtype])
    z[:, 50:] = torch.finfo(TYPES[dtype]).min
    ids, teacher = r.integers(0, 50, (n, 7)), r.normal(size=(n, 7))
    ids[0, 2] = 60
    ids[1, 3:] = [50, 70, 80, 299]
    ids[2] = r.integers(50, v, 7)                # the weights' sum is rounded, the loss is not to be beyond it
    ids[3], teacher[3] = 77, -200.0 * np.arange(7)        # all of the weight on one
    ids[4, :3], teacher[4, 3:] = 90, -np.inf
    weights = np.full(n, 0.5)
    d_teacher = on_gpu(teacher, torch.float32)
    want, ref, size = O.distill(f64(z), ids, f64(d_teacher), temperature, weights)
    losses, grad = gpu.distill_step(z, on_gpu(ids, torch.int64), d_teacher, on_gpu(weights, torch.float32), temperature)
    _all_near(losses, want)
    near(grad, ref, size, dtype)
    z.requires_grad_()
    loss = gpu.distill_loss(z, on_gpu(ids, torch.int32), d_teacher, temperature)
    _all_near(loss, want)
    if temperature > 0.95:
        assert torch.isfinite(losses).all() and torch.isfinite(loss).all()
    dz, = torch.autograd.grad(loss, z, on_gpu(weights, torch.float32))
    near(dz, ref, size, dtype)


# How far rounding goes on the whole.  A row's sum: a thread's terms are added up 4 to 32 at a time and these sums, some 25 here, one
# after the other; log Z has a value of up to 16, of which half a unit is 4.8e-7, as the difference to it has, and the terms' own
# exponents, up to 24 to the base 2, are rounded by up to 9.5e-7, independently for the hundreds of terms that a sum comes from.
# Uniform errors of half a unit have a root mean square of half a unit / sqrt(3): 2.8e-7 twice, and the rest below that: 4.8e-7.
@pytest.mark.parametrize("dtype,temperature", [("f16", 1.0), ("f32", 0.7), ("bf16", 1.0)])
@pytest.mark.parametrize("top", [0, 5])
def test_rounding_of_long_rows(gpu, dtype, temperature, top):
    n, v = 4096, 50_001
    z = (2.5 * torch.randn(n, v, device="cuda")).to(TYPES[dtype])
    targets = torch.randint(0, v, (n,), device="cuda")
    z[torch.arange(n, device="cuda"), targets] += (12 * torch.rand(n, device="cuda")).to(z.dtype)
    z.requires_grad_()
    got = gpu.token_logprobs(z, targets, top, temperature)
    g = torch.randn(n, device="cuda")
    dz, = torch.autograd.grad(got[0], z, g)
    lp_off = h_off = off = size = 0.0
    for a in range(0, n, 512):
        logp = torch.log_softmax(z[a:a + 512].detach().double() / temperature, 1)
        t = targets[a:a + 512, None]
        lp_off += (got[0][a:a + 512].double() - logp.gather(1, t)[:, 0]).square().sum().item()
        p = torch.exp(logp)
        h_off += (got[1][a:a + 512].double() + (p * logp).sum(1)).square().sum().item()
        want = -p.scatter_add(1, t, -torch.ones_like(t, dtype=torch.float64)) * (g[a:a + 512, None].double() / temperature)
        off += (dz[a:a + 512].double() - want).square().sum().item()
        size += want.square().sum().item()
    assert (lp_off / n) ** 0.5 < 4.8e-7 and (h_off / n) ** 0.5 < 4.8e-7
    # a gradient's largest terms, which its size comes from, have exponents below 4, of which half a unit is 1.2e-7 or less, twice
    # (the product, the factor's own rounding); an exponential's, a sum's, a factor's and the result's roundings are 6e-8 each
    if dtype == "f32":
        assert (off / size) ** 0.5 < 2.0e-7


# In a gradient from statistics the sum itself is a factor: the rounding of its logarithm (half a unit of 16 to 32 is 9.5e-7) has no part in it.
@pytest.mark.parametrize("n,v", [(3, 262_145), (2000, 100_000), (200, 50_001)])
def test_gradients_of_flat_rows(gpu, n, v):
    """Logits alike: every term is 1 and every gradient is 1 / v, to four roundings and those of the sum (of whole numbers: none)."""
    z = torch.full((n, v), 2.5, device="cuda", requires_grad=True)
    ids, teacher = torch.zeros(n, 1, dtype=torch.int64, device="cuda"), torch.zeros(n, 1, device="cuda")
    lp, _ = gpu.token_logprobs(z, ids[:, 0])
    by_logp, = torch.autograd.grad(lp.sum(), z)
    by_loss, = torch.autograd.grad(gpu.distill_loss(z, ids, teacher).sum(), z)
    _, by_step = gpu.distill_step(z.detach(), ids, teacher)
    for dz in (-by_logp, by_loss, by_step):
        assert ((dz[:, 1:].double() * v - 1).abs() <= 4 * 2.0 ** -24).all()


@pytest.mark.parametrize("v", [50, 20_000, 140_000])
def test_distillation_of_a_small_weight_at_a_high_temperature(gpu, v):
    """A weight of 4e-31 over a temperature of 1e20 is 0 in 32 bits; times a token that is ruled out it is not to be NaN."""
    z = torch.randn(2, v, device="cuda")
    z[0, 7] = -float("inf")
    ids, teacher = torch.tensor([[3, 7], [3, 7]], device="cuda"), torch.tensor([[0.0, -7e21], [0.0, -7e21]], device="cuda")
    want = O.distill(f64(z), ids.cpu().numpy(), f64(teacher), float(np.float32(1e20)), np.ones(2))[0]
    assert want[0] == np.inf
    near_abs(gpu.distill_loss(z, ids, teacher, 1e20), want, 2 * SUM)
    near_abs(gpu.distill_step(z, ids, teacher, temperature=1e20)[0], want, 2 * SUM)


# ---- derivatives that are not formed -----------------------------------------------------
def test_tangents_of_forward_mode_are_refused(gpu):
    import torch.autograd.forward_ad as forward
    z, t = torch.randn(4, 9, device="cuda"), torch.zeros(4, dtype=torch.int64, device="cuda")
    ids, teacher, ones = torch.zeros(4, 3, dtype=torch.int64, device="cuda"), torch.zeros(4, 3, device="cuda"), torch.ones(4, device="cuda")
    with forward.dual_level():
        def dual(x):
            return forward.make_dual(x, torch.ones_like(x))
        for call in (lambda: gpu.embed(dual(z), t), lambda: gpu.embed(dual(z.clone().requires_grad_()), t), lambda: gpu.embed_grad(dual(z), t, 5),
                     lambda: gpu.embed_grad(z, t, 5, out=dual(torch.zeros(5, 9, device="cuda"))), lambda: gpu.token_logprobs(dual(z), t),
                     lambda: gpu.token_logprobs(dual(z), t, 3), lambda: gpu.distill_loss(dual(z), ids, teacher), lambda: gpu.distill_loss(z, ids, dual(teacher)),
                     lambda: gpu.distill_step(dual(z), ids, teacher), lambda: gpu.distill_step(z, ids, dual(teacher)),
                     lambda: gpu.distill_step(z, ids, teacher, dual(ones)), lambda: gpu.distill_step(z, ids, teacher, out=dual(torch.zeros_like(z)))):
            with pytest.raises(RuntimeError, match="forward mode"):
                call()
        # without one they compute as ever
        assert torch.equal(gpu.embed(z, t), z[t]) and gpu.token_logprobs(z, t)[0].shape == (4,)


def test_tangents_of_a_gradient_are_refused(gpu):
    import torch.autograd.forward_ad as forward
    z, t = torch.randn(4, 9, device="cuda", requires_grad=True), torch.zeros(4, dtype=torch.int64, device="cuda")
    ids, teacher = torch.zeros(4, 3, dtype=torch.int64, device="cuda"), torch.zeros(4, 3, device="cuda")
    with forward.dual_level():
        for out in (gpu.embed(z, t), gpu.token_logprobs(z, t)[0], gpu.distill_loss(z, ids, teacher)):
            with pytest.raises(RuntimeError, match="forward mode"):
                torch.autograd.grad(out, z, forward.make_dual(torch.ones_like(out), torch.ones_like(out)))


def test_embed_grad_forms_no_graph(gpu):
    grad, ids = torch.randn(4, 9, device="cuda", requires_grad=True), torch.zeros(4, dtype=torch.int64, device="cuda")
    with pytest.raises(ValueError, match="detach"):
        gpu.embed_grad(grad, ids, 5)
    with pytest.raises(ValueError, match="detach"):
        gpu.embed_grad(grad * 2, ids, 5, out=torch.zeros(5, 9, device="cuda"))
    want = gpu.embed_grad(grad.detach(), ids, 5)
    with torch.no_grad():
        assert torch.equal(gpu.embed_grad(grad, ids, 5), want)


def test_distillation_into_what_requires_a_gradient(gpu):
    z, ids, teacher = torch.randn(4, 9, device="cuda"), torch.randint(0, 9, (4, 3), device="cuda"), torch.randn(4, 3, device="cuda")
    want = gpu.distill_step(z, ids, teacher)[1]
    leaf, weight = z.clone().requires_grad_(), torch.eye(9, device="cuda", requires_grad=True)
    for logits, out in ((leaf, leaf), (z, leaf), (z, torch.zeros(4, 9, device="cuda", requires_grad=True)), (z, z @ weight), (z @ weight, z @ weight)):
        before = out.detach().clone()
        with pytest.raises(ValueError, match="out must not require a gradient"):
            gpu.distill_step(logits, ids, teacher, out=out)
        assert torch.equal(out, before)
    # a model's own logits give way to their gradient, which goes on to its weights
    logits = z @ weight
    _, dz = gpu.distill_step(logits, ids, teacher, out=logits)
    assert dz is logits and torch.equal(dz, want)
    by_weight, = torch.autograd.grad(logits, weight, dz.detach())
    assert torch.allclose(by_weight, z.t() @ want, atol=1e-5)
    with torch.no_grad():
        assert torch.equal(gpu.distill_step(leaf, ids, teacher, out=leaf)[1], want)


@pytest.mark.parametrize("shape", [(3, 5, 700), (2, 40, 9001)])
def test_next_tokens_of_a_batch(gpu, shape):
    """Logits without their last position are at two distances; all of them with ids of -1 there are the same."""
    b, t, v = shape
    z = torch.randn(shape, device="cuda")
    tokens, g = torch.randint(0, v, (b, t), device="cuda"), torch.randn(b, t - 1, device="cuda")
    ids, teacher = torch.randint(0, v, (b, t, 4), device="cuda"), torch.randn(b, t, 4, device="cuda")
    for call in (lambda: gpu.token_logprobs(z[:, :-1], tokens[:, 1:]), lambda: gpu.distill_loss(z[:, :-1], ids[:, :-1], teacher[:, :-1]),
                 lambda: gpu.distill_step(z[:, :-1], ids[:, :-1], teacher[:, :-1])):
        with pytest.raises(ValueError, match="ids of -1"):
            call()
    targets = torch.cat([tokens[:, 1:], torch.full_like(tokens[:, :1], -1)], 1)
    ids[:, -1] = -1
    whole, cut = z.clone().requires_grad_(), z[:, :-1].contiguous().requires_grad_()
    for a, c in ((gpu.token_logprobs(whole, targets)[0], gpu.token_logprobs(cut, tokens[:, 1:])[0]),
                 (gpu.distill_loss(whole, ids, teacher), gpu.distill_loss(cut, ids[:, :-1], teacher[:, :-1]))):
        assert (a[:, -1] == 0).all()
        near_abs(a[:, :-1], f64(c), SUM)
        by_whole, = torch.autograd.grad(a[:, :-1], whole, g)
        by_cut, = torch.autograd.grad(c, cut, g)
        assert (by_whole[:, -1] == 0).all()
        near(by_whole[:, :-1], f64(by_cut), np.abs(f64(by_cut)) + np.abs(f64(g))[:, :, None] * 1e-3, "f32", 2 * SUM)


# ---- many tokens: pieces of rows, joined, added to what is there ---------------------------
def _many(gpu, ids, d, v, dtype, scale=0.5):
    """The gradient of more tokens than one launch takes, written and added to a float32 and to an own-type gradient."""
    ids = on_gpu(ids, torch.int64)
    assert ids.numel() > 4096
    grad = torch.randn(ids.numel(), d, device="cuda").to(TYPES[dtype])
    valid = (ids >= 0) & (ids < v)
    want = torch.zeros(v, d, dtype=torch.float64, device="cuda").index_add_(0, ids[valid], grad[valid].double() * scale)
    size = torch.zeros(v, d, dtype=torch.float64, device="cuda").index_add_(0, ids[valid], grad[valid].double().abs() * scale)
    count = torch.bincount(ids[valid], minlength=v).double()[:, None]
    got = gpu.embed_grad(grad, ids, v, scale)
    # an addition for each token, the factor, the sum with what is there: 2^-24 each; and one rounding to the type
    far = (got.double() - want).abs() - HALF_UNIT[dtype] * want.abs() * 1.01 - LEAST[dtype] - (count + 2) * 2.0 ** -24 * size
    assert (far <= 0).all()
    assert torch.equal(got, gpu.embed_grad(grad, ids.int(), v, scale))
    none = count[:, 0] == 0
    assert not got[none].any()
    for kind in {dtype, "f32"}:
        base = torch.randn(v, d, device="cuda").to(TYPES[kind])
        into = gpu.embed_grad(grad, ids, v, scale, out=base.clone())
        sum_ = want + base.double()
        far = (into.double() - sum_).abs() - HALF_UNIT[kind] * sum_.abs() * 1.01 - LEAST[kind] - (count + 3) * 2.0 ** -24 * (size + base.double().abs())
        assert (far <= 0).all() and torch.equal(into[none], base[none])
    return got


# Pieces have 8 tokens (below 2^21 elements in all) or 16; rows of more than 16 pieces are joined by groups.
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("d", [20, 100, 513])
@pytest.mark.parametrize("counts", [[7, 8, 9, 15, 16, 17], [1, 31, 32, 33, 2, 127, 128, 129], [128, 1, 255, 256, 257, 136, 137], [2000, 1, 4096, 3]])
def test_lookup_gradient_by_pieces(gpu, dtype, d, counts):
    r = gen(d + sum(counts))
    rows = np.repeat(np.arange(len(counts)), counts)
    ids = np.concatenate([rows, r.integers(len(counts), 4000, max(4100, 5000 - len(rows)))])      # others, a few tokens each
    n = len(ids)
    assert (n * 20 < 1 << 21) and (n * 513 >= 1 << 21)
    _many(gpu, ids, d, 4003, dtype)                        # the counted rows' tokens next to one another, from the first on
    _many(gpu, r.permutation(ids), d, 4003, dtype)
    _many(gpu, 4002 - ids, d, 4003, dtype)                 # the last rows of the table


def test_lookup_gradient_of_a_million_tokens(gpu):
    """More chunks of tokens than a wavefront looks at at a time, by few rows and by many."""
    r = gen(17)
    n = 1_100_001
    for v, d, dtype in ((300, 3, "f32"), (70_000, 4, "bf16"), (2_200_000, 2, "f16")):
        ids = np.where(np.arange(n) % 11 == 3, v // 3, r.integers(-1, v + 1, n))
        _many(gpu, ids, d, v, dtype)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("n,v,d", [(1, 1, 1), (33, 5, 100), (700, 2500, 1025), (4096, 300, 40)])
def test_lookup_gradient_of_few_tokens_added_to_its_own_type(gpu, dtype, n, v, d):
    r = gen(n + v)
    ids = r.integers(-1, v + 1, n)
    grad = on_gpu(r.normal(size=(n, d)), TYPES[dtype])
    want, size, count = O.embed_grad(f64(grad), ids, v, 0.5)
    base = torch.randn(v, d, device="cuda").to(TYPES[dtype])
    into = gpu.embed_grad(grad, on_gpu(ids, torch.int64), v, 0.5, out=base.clone())
    near(into, want + f64(base), size + np.abs(f64(base)), dtype, (count[:, None] + 3) * 2.0 ** -24)
    assert torch.equal(into[on_gpu(count == 0, torch.bool)], base[on_gpu(count == 0, torch.bool)])


@pytest.mark.parametrize("n,v,d,dtype", [(9000, 700, 96, "bf16"), (5000, 90_000, 12, "f32")])
def test_graph_of_the_gradient_of_many_tokens(gpu, n, v, d, dtype):
    """Recorded and replayed: the launches that group, clear, sum and join, on other tokens each time."""
    grad, ids = torch.randn(n, d, device="cuda").to(TYPES[dtype]), torch.randint(0, v, (n,), device="cuda")
    total = torch.zeros(v, d, device="cuda")

    def work():
        return gpu.embed_grad(grad, ids, v, 0.5), gpu.embed_grad(grad, ids, v, 2.0, out=total)

    work()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = work()
    for i in range(4):
        ids.copy_(torch.randint(-1, v, (n,), device="cuda") if i % 2 else torch.randint(0, 20, (n,), device="cuda"))
        grad.copy_(torch.randn(n, d, device="cuda"))
        total.copy_(torch.randn(v, d, device="cuda"))
        before = total.clone()
        want = [x.clone() for x in work()]
        total.copy_(before)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want)), i
