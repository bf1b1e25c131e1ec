"""Verification of drafted tokens against 64 bits, and that what it draws is distributed as the model says."""
import math

import numpy as np
import pytest
import torch

import recurrent_oracles as O

pytestmark = pytest.mark.gpu
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def inputs(n, k, v, slots, dtype, seed=0, likely=0.7, spread=2.0):
    g = torch.Generator().manual_seed(seed)
    z = spread * torch.randn(n, k + 1, v, generator=g)
    best = z.argmax(2)
    drafts = torch.where(torch.rand(n, k, generator=g) < likely, best[:, :k], torch.randint(0, v, (n, k), generator=g))
    drafts[torch.rand(n, k, generator=g) < 0.05] = -1
    ids = teacher = None
    if slots:
        ids = torch.randint(0, v, (n, k, slots), generator=g)
        ids[:, :, 0] = drafts.clamp(min=0)
        ids[:, :, slots // 2] = ids[:, :, 0]                 # the draft in two slots
        ids[torch.rand(n, k, slots, generator=g) < 0.1] = -1
        teacher = 2.0 * torch.randn(n, k, slots, generator=g)
        teacher[torch.rand(n, k, slots, generator=g) < 0.1] = -math.inf
    return z.to(TYPES[dtype]), drafts, torch.rand(n, k + 1, generator=g), ids, teacher


def check(gpu, z, drafts, u, ids=None, teacher=None, temperature=1.0, wide=True, on_border=False):
    whole = lambda t: None if t is None else (t if wide else t.int()).cuda()          # noqa: E731
    got = gpu.verify_drafts(z.cuda(), whole(drafts), u.cuda(), whole(ids), None if teacher is None else teacher.cuda(), temperature)
    num = lambda t: None if t is None else t.double().numpy()                         # noqa: E731
    tokens, accepted, logps, near = O.verify(num(z), drafts.numpy(), num(u), None if ids is None else ids.numpy(), num(teacher), float(np.float32(temperature)))
    # (both sides are off by 1e-12 at most; inputs that come nearer to a border than that say nothing)
    assert near > 1e-11 or on_border
    assert got[0].dtype == torch.int32 and got[1].dtype == torch.int32 and got[2].dtype == torch.float32
    assert torch.equal(got[0].cpu(), torch.from_numpy(tokens).int()) and torch.equal(got[1].cpu(), torch.from_numpy(accepted).int())
    mine, want = got[2].cpu().numpy(), logps
    assert (np.isnan(mine) == np.isnan(want)).all()
    some = ~np.isnan(want)
    assert (np.abs(mine[some] - want[some]) <= O.STEP * np.abs(want[some]) * (1 + 1e-6) + 1e-11).all()
    return got


SIZES = [(1, 0, 1), (3, 0, 9), (1, 1, 2), (5, 3, 17), (4, 4, 2047), (3, 2, 2048), (2, 7, 2049), (9, 5, 1000), (2, 3, 50_001), (1, 2, 131_072), (2, 256, 33), (40, 2, 4096)]


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("slots", [0, 1, 5, 64])
@pytest.mark.parametrize("size", SIZES, ids=str)
def test_against_64_bits(gpu, size, slots, dtype):
    n, k, v = size
    z, drafts, u, ids, teacher = inputs(n, k, v, slots if k else 0, dtype, seed=slots)
    check(gpu, z, drafts, u, ids, teacher, wide=slots != 5)


@pytest.mark.parametrize("temperature", [0.1, 0.7, 3.0, 1e4])
def test_temperatures(gpu, temperature):
    z, drafts, u, ids, teacher = inputs(20, 4, 777, 6, "bf16", seed=3)
    check(gpu, z, drafts, u, ids, teacher, temperature)
    check(gpu, z, drafts, u, temperature=temperature)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("temperature", [1e-29, 1e-3, 1.0, 1e3, 1e29])
def test_rows_of_all_magnitudes(gpu, temperature, dtype):
    """Some stretches of a row beyond what powers of 2 in 64 bits reach, up or down, others not; all of it shifted; nothing but that."""
    z, drafts, u, ids, teacher = inputs(8, 2, 9000, 6, "f32", seed=21)
    z[0, :, :2048] += 2000.0
    z[1, :, 2048:5000] -= 2000.0
    z[2, :, :] -= 700.0
    z[3, :, 4096:] += 600.0
    z[4, :, :4096] = -math.inf
    z[5] += 3000.0
    z[6] -= 3000.0
    z[7, :, 3000:] = -math.inf
    z[7, :, :2048] -= 630.0
    z = (z * temperature).clamp(-3e38, 3e38).to(TYPES[dtype])
    check(gpu, z, drafts, u, ids, teacher, temperature, on_border=True)
    check(gpu, z, drafts, u, temperature=temperature, on_border=True)


@pytest.mark.parametrize("slots", [200, 1023, 1024])
@pytest.mark.parametrize("teacher_type", ["f32", "f16", "bf16"])
def test_many_slots(gpu, slots, teacher_type):
    z, drafts, u, ids, teacher = inputs(6, 3, 300, slots, "f16", seed=slots)
    check(gpu, z, drafts, u, ids, teacher.to(TYPES[teacher_type]))


def test_masked_logits(gpu):
    """Ruled out by -inf or the type's lowest value, all but one, all."""
    for dtype in TYPES.values():
        z, drafts, u, ids, teacher = inputs(8, 3, 5000, 4, "f32", seed=11)
        z = z.to(dtype)
        z[0, :, ::2] = -math.inf
        z[1, :, 100:] = -math.inf
        z[2, :, 1:] = -math.inf
        z[3, :, :-1] = torch.finfo(dtype).min
        z[4, 1] = -math.inf
        z[5, 0, 77] = math.nan
        z[6, 2, 4999] = math.inf
        z[7] = torch.finfo(dtype).min
        drafts = drafts.clamp(min=0)
        check(gpu, z, drafts, u, ids, teacher)
        check(gpu, z, drafts, u)


def test_teachers_that_say_nothing(gpu):
    z, drafts, u, ids, teacher = inputs(7, 2, 400, 5, "f32", seed=12)
    drafts = drafts.clamp(min=0)
    ids[0] = -1                                       # no slot filled: whatever the model holds for possible stands
    teacher[1] = -math.inf
    ids[2] = 401                                      # all beyond the vocabulary
    ids[3, :, 2:] = 1 << 40
    teacher[4, 0, 1], ids[4, 0, 1] = math.nan, 3
    teacher[5, 1, 1], ids[5, 1, 1] = math.inf, 3
    teacher[6, :, 1], ids[6, :, 1] = math.nan, -1     # an empty slot's logit is not looked at
    check(gpu, z, drafts, u, ids, teacher)


def test_drafts_beyond_the_vocabulary(gpu):
    z, drafts, u, _, _ = inputs(4, 3, 100, 0, "f32", seed=13)
    drafts[0, 0], drafts[1, 1], drafts[2, 2] = 100, 1 << 40, 2 ** 31
    u[:2, :3] = 0.0
    check(gpu, z, drafts, u)
    u[:] = -1.0                                       # not a random number of [0, 1): nothing is read beyond the row all the same
    got = gpu.verify_drafts(z.cuda(), drafts.cuda(), u.cuda())
    assert (got[0] < 100).all()


def test_borders_of_the_random_numbers(gpu):
    z, drafts, u, ids, teacher = inputs(6, 2, 3000, 3, "f32", seed=14)
    u[0], u[1, 2], u[2, 2], u[3] = 0.0, 1.0 - 2.0 ** -24, 0.0, 1.0 - 2.0 ** -24
    u[4, 2], u[5, 0] = math.nan, math.nan
    check(gpu, z, drafts, u, ids, teacher)
    check(gpu, z, drafts, u)
    z[:, :, -1500:] = -math.inf                       # the last that can be drawn is far from the end
    u[:, 2] = 1.0
    check(gpu, z, drafts, u)


def test_certain_drafts_of_a_certain_model(gpu):
    """p = q = 1: kept with any number below 1; with 1 nothing is left but p itself."""
    z = torch.full((3, 2, 50), -math.inf)
    z[:, :, 7] = 3.0
    drafts = torch.tensor([[7], [7], [8]])
    u = torch.tensor([[1.0 - 2.0 ** -24, 0.5], [1.0, 0.5], [0.0, 0.9]])
    got = check(gpu, z, drafts, u, on_border=True)      # (1 < 1 is one)
    assert got[0].tolist() == [[7, 7], [7, -1], [7, -1]]


def test_rows_at_a_distance(gpu):
    for dtype, cut in (("bf16", 1), ("f16", 3), ("f32", 1)):
        z, drafts, u, ids, teacher = inputs(5, 3, 2500, 4, dtype, seed=15)
        wide = torch.cat([z, z], 2).cuda()[:, :, cut:2500 + cut]
        want = gpu.verify_drafts(wide.contiguous(), drafts.cuda(), u.cuda(), ids.cuda(), teacher.cuda())
        got = gpu.verify_drafts(wide, drafts.cuda().t().contiguous().t(), torch.stack([u, u], 2).cuda()[:, :, 0], ids.cuda(), teacher.cuda())
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_distribution(gpu):
    """400 000 sequences with one draft from q: tokens are distributed as p says, whatever q is."""
    n, v = 400_000, 12
    g = torch.Generator(device="cuda").manual_seed(5)
    z = torch.randn(1, 2, v, generator=g, device="cuda").expand(n, 2, v).contiguous()
    p = torch.softmax(z[0].double(), 1)
    for certain in (False, True):
        ids = torch.randint(0, v, (1, 1, 5), generator=g, device="cuda").expand(n, 1, 5).contiguous()
        teacher = torch.randn(1, 1, 5, generator=g, device="cuda").expand(n, 1, 5).contiguous()
        slot = torch.multinomial(torch.softmax(teacher[0, 0], 0), n, replacement=True, generator=g)
        drafts = ids[0, 0][slot][:, None] if not certain else torch.full((n, 1), int(p[0].argmax()), device="cuda")
        u = torch.rand(n, 2, generator=g, device="cuda")
        tokens, accepted, _ = gpu.verify_drafts(z, drafts, u, *(() if certain else (ids, teacher)))
        got = torch.bincount(tokens[:, 0].long(), minlength=v).double() / n
        # six standard deviations of each share
        assert ((got - p[0]).abs() < 6 * (p[0] * (1 - p[0]) / n).sqrt()).all()
        second = tokens[accepted == 1, 1].long()
        m = len(second)
        got = torch.bincount(second, minlength=v).double() / m
        # (the last number draws the second token only where it did not draw the first)
        assert ((got - p[1]).abs() < 6 * (p[1] * (1 - p[1]) / m).sqrt()).all()


def test_sampling_without_drafts(gpu):
    n, v = 300_000, 30
    g = torch.Generator(device="cuda").manual_seed(6)
    z = torch.randn(1, 1, v, generator=g, device="cuda").expand(n, 1, v).contiguous()
    tokens, accepted, logp = gpu.verify_drafts(z, torch.zeros(n, 0, dtype=torch.int64, device="cuda"), torch.rand(n, 1, generator=g, device="cuda"))
    p = torch.softmax(z[0, 0].double(), 0)
    got = torch.bincount(tokens[:, 0].long(), minlength=v).double() / n
    assert not accepted.any() and ((got - p).abs() < 6 * (p * (1 - p) / n).sqrt()).all()
    assert (logp[:, 0].double() - p.log()[tokens[:, 0].long()]).abs().max() < 1e-6


def test_drafts_from_a_models_best(gpu):
    """What `token_logprobs` returns for alternatives is a distribution to draw drafts from."""
    g = torch.Generator(device="cuda").manual_seed(7)
    z = torch.randn(16, 4, 3000, generator=g, device="cuda")
    small = z[:, :3] + 0.5 * torch.randn(16, 3, 3000, generator=g, device="cuda")
    _, _, ids, logp = gpu.token_logprobs(small, torch.zeros(16, 3, dtype=torch.int64, device="cuda"), top=20)
    slot = torch.multinomial(torch.softmax(logp, 2).flatten(0, 1), 1, generator=g).view(16, 3, 1)
    drafts = ids.gather(2, slot)[:, :, 0]
    u = torch.rand(16, 4, generator=g, device="cuda")
    got = gpu.verify_drafts(z, drafts, u, ids, logp)
    want = O.verify(z.double().cpu().numpy(), drafts.cpu().numpy(), u.double().cpu().numpy(), ids.cpu().numpy(), logp.double().cpu().numpy(), 1.0)
    assert np.array_equal(got[0].cpu().numpy(), want[0]) and np.array_equal(got[1].cpu().numpy(), want[1])


def test_large_vocabulary(gpu):
    """More chunks than a workgroup has threads."""
    g = torch.Generator(device="cuda").manual_seed(8)
    v = 2_000_003
    z = torch.randn(2, 2, v, generator=g, device="cuda").half()
    drafts, u = torch.tensor([[5], [v - 1]], device="cuda"), torch.tensor([[0.9, 0.3], [0.9, 0.99999]], device="cuda")
    tokens, accepted, _ = gpu.verify_drafts(z, drafts, u)
    p = torch.softmax(z[:, 0].double(), 1)
    p[0, 5], p[1, v - 1] = 0.0, 0.0
    sums = torch.cumsum(p, 1)
    want = torch.searchsorted(sums, (u[:, 1:].double() * sums[:, -1:]), right=True)[:, 0]
    assert not accepted.any() and torch.equal(tokens[:, 0].long(), want)


def test_recorded_and_replayed(gpu):
    z, drafts, u, ids, teacher = (t.cuda() for t in inputs(7, 3, 5000, 5, "bf16", seed=16))
    gpu.verify_drafts(z, drafts, u, ids, teacher)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = gpu.verify_drafts(z, drafts, u, ids, teacher)
    for turn in range(4):
        z.normal_(0.0, 3.0)
        u.uniform_()
        drafts.random_(-1, 5000)
        want = gpu.verify_drafts(z, drafts, u, ids, teacher)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want)), turn


def test_refusals(gpu):
    z, drafts, u, ids, teacher = (t.cuda() for t in inputs(2, 3, 50, 4, "f32"))
    for bad, error in [
        (lambda: gpu.verify_drafts(z.double(), drafts, u), TypeError), (lambda: gpu.verify_drafts(z[0], drafts, u), ValueError),
        (lambda: gpu.verify_drafts(z, drafts[:, :2], u), ValueError), (lambda: gpu.verify_drafts(z, drafts.float(), u), TypeError),
        (lambda: gpu.verify_drafts(z, drafts, u[:, :3]), ValueError), (lambda: gpu.verify_drafts(z, drafts, u.double()), TypeError),
        (lambda: gpu.verify_drafts(z, drafts, u, ids), ValueError), (lambda: gpu.verify_drafts(z, drafts, u, None, teacher), ValueError),
        (lambda: gpu.verify_drafts(z, drafts, u, ids, teacher[:, :, :3]), ValueError), (lambda: gpu.verify_drafts(z, drafts, u, ids[:, :2], teacher[:, :2]), ValueError),
        (lambda: gpu.verify_drafts(z, drafts, u, ids[:, :, :0], teacher[:, :, :0]), ValueError), (lambda: gpu.verify_drafts(z, drafts, u, temperature=0.0), ValueError),
        (lambda: gpu.verify_drafts(z, drafts, u, temperature=float("nan")), ValueError), (lambda: gpu.verify_drafts(z.transpose(1, 2), drafts, u), ValueError),
        (lambda: gpu.verify_drafts(z.clone().requires_grad_(), drafts, u), ValueError), (lambda: gpu.verify_drafts(z, drafts.cpu(), u), TypeError),
        (lambda: gpu.verify_drafts(torch.zeros(1, 258, 5, device="cuda"), torch.zeros(1, 257, dtype=torch.int64, device="cuda"), torch.zeros(1, 258, device="cuda")), ValueError),
    ]:
        with pytest.raises(error):
            bad()
    assert gpu.verify_drafts(z[:0], drafts[:0], u[:0])[0].shape == (0, 4)
