"""Norms of gradients and clipping against 64 bits."""
import math

import numpy as np
import pytest
import torch

import recurrent_oracles as O

pytestmark = pytest.mark.gpu
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def tensors(shapes, dtype, seed=0, size=1.0):
    g = torch.Generator().manual_seed(seed)
    types = [TYPES[dtype]] * len(shapes) if dtype in TYPES else [list(TYPES.values())[i % 3] for i in range(len(shapes))]
    return [(size * torch.randn(s, generator=g)).to(t).cuda() for s, t in zip(shapes, types)]


def doubles(ts):
    return [t.double().cpu().numpy() for t in ts]


def close(got, want, dtype):
    """The factor is rounded to 32 bits, the product once there and once to its type."""
    half = torch.finfo(dtype).eps / 2
    bound = (2 * O.STEP + half * (1 + 2 * O.STEP)) * np.abs(want) + (2.0 ** -25 if dtype == torch.float16 else 2.0 ** -127)
    assert (np.abs(got.double().cpu().numpy() - want) <= bound).all()


SHAPES = [
    [(1,)], [()], [(7,), (1, 1)], [(2048,)], [(2049,), (0,), (5, 3)], [(100, 333), (17,), (4096, 5), (1,)], [(3, 5, 7, 11)] * 5,
    [(i % 97 + 1,) for i in range(300)], [(70_001, 9), (2, 2)], [(600, 1000)] * 3 + [(13,)] * 130,
]


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16", "mixed"])
@pytest.mark.parametrize("which", range(len(SHAPES)))
def test_norm_and_clip(gpu, which, dtype):
    grads = tensors(SHAPES[which], dtype)
    for scale in (1.0, -0.5, 2.0 ** -12):
        want = O.norm(doubles(grads), scale)
        got = gpu.grad_norm(grads, scale)
        # sums in 64 bits, one rounding
        assert got.shape == () and got.dtype == torch.float32 and abs(got.item() - want) <= (1 + 1e-6) * O.STEP * want + 1e-45
        for share in (0.25, 4.0):
            norm, clipped = O.clip(doubles(grads), want * share, scale)
            for kind in ("place", "same", "f32"):
                mine = [g.clone() for g in grads]
                out = None if kind == "place" else [torch.full_like(g, 7.0, dtype=torch.float32 if kind == "f32" else g.dtype) for g in grads]
                n = gpu.clip_grads(mine, want * share, scale, out=out)
                assert torch.equal(n, got)
                for a, b, g in zip(out or mine, clipped, grads):
                    close(a, b, a.dtype)
                if kind != "place":
                    assert all(torch.equal(a, b) for a, b in zip(mine, grads))
                elif share > 1 and scale == 1.0:
                    assert all(torch.equal(a, b) for a, b in zip(mine, grads))


def test_parts_of_one_buffer(gpu):
    """Neighbours at odd places, all but one element of which belong to the call: nothing beside them is written."""
    sizes = [1, 3, 2047, 2049, 5, 40_003, 8, 1]
    for dtype in TYPES.values():
        flat = torch.randn(sum(sizes) + 2).to(dtype).cuda()
        before = flat.clone()
        parts = list(flat[1:-1].split(sizes))
        norm = gpu.clip_grads(parts[:4] + parts[5:], 1.0)
        want, _ = O.clip(doubles([before[1:-1].split(sizes)[i] for i in (0, 1, 2, 3, 5, 6, 7)]), 1.0, 1.0)
        assert abs(norm.item() - want) <= 2 * O.STEP * want
        hole = slice(1 + sum(sizes[:4]), 1 + sum(sizes[:5]))
        assert flat[0] == before[0] and flat[-1] == before[-1] and torch.equal(flat[hole], before[hole])
        close(flat[1:hole.start], before[1:hole.start].double().cpu().numpy() / want, dtype)


def test_orders_of_dimensions(gpu):
    g = torch.randn(30, 50, device="cuda").t()
    h = torch.randn(4, 6, 5, 3, device="cuda").contiguous(memory_format=torch.channels_last)
    want, clipped = O.clip(doubles([g, h]), 2.0, 1.0)
    gpu.clip_grads([g, h], 2.0)
    for a, b in zip((g, h), clipped):
        close(a, b, torch.float32)


@pytest.mark.parametrize("dtype, size", [("f32", 1e30), ("f32", 1e-30), ("bf16", 1e37), ("bf16", 1e-38), ("f16", 3e4), ("f16", 1e-7)])
def test_large_and_small_values(gpu, dtype, size):
    """Whose squares 32 bits do not hold."""
    grads = tensors([(5000,), (33, 7)], dtype, size=size)
    grads = [g.clamp(-torch.finfo(g.dtype).max, torch.finfo(g.dtype).max) for g in grads]
    want, clipped = O.clip(doubles(grads), 1.0, 1.0)
    norm = gpu.clip_grads(grads, 1.0)
    # (5000 values of 1e37 have a norm beyond 32 bits: infinite, and clipping nothing)
    assert (want == norm.item() == math.inf) == ((dtype, size) == ("bf16", 1e37)) and (want == norm.item() or abs(norm.item() - want) <= 2 * O.STEP * want)
    for a, b in zip(grads, clipped):
        close(a, b, a.dtype)


def test_norms_that_are_no_number(gpu):
    for bad in (float("nan"), float("inf"), -float("inf")):
        grads = [torch.randn(3000, device="cuda"), torch.randn(5, device="cuda", dtype=torch.bfloat16)]
        grads[0][1234] = bad
        before = [g.clone() for g in grads]
        norm = gpu.clip_grads(grads, 0.1)
        assert math.isnan(norm.item()) if bad != bad else norm.item() == float("inf")
        assert all(torch.equal(a.nan_to_num(7.0), b.nan_to_num(7.0)) for a, b in zip(grads, before))
        gpu.clip_grads(grads, 0.1, scale=0.5)
        assert all(torch.equal((0.5 * b).nan_to_num(7.0), a.nan_to_num(7.0)) for a, b in zip(grads, before))


def test_nothing_to_clip(gpu):
    assert gpu.grad_norm([]).item() == 0.0 and gpu.clip_grads([], 1.0).item() == 0.0
    empty = torch.zeros(0, 5, device="cuda")
    assert gpu.grad_norm([empty]).item() == 0.0 and gpu.clip_grads([empty], 1.0).item() == 0.0
    zeros = [torch.zeros(70_000, device="cuda")]
    assert gpu.clip_grads(zeros, 0.0).item() == 0.0 and not zeros[0].any()
    ones = [torch.ones(100, device="cuda")]
    assert gpu.clip_grads(ones, 0.0).item() == 10.0 and not ones[0].any()
    ones = [torch.ones(100, device="cuda")]
    assert gpu.clip_grads(ones, float("inf"), 2.0).item() == 20.0 and (ones[0] == 2).all()


def test_many_tensors_take_many_tables(gpu):
    """More than a launch's table holds; the order of the list does not matter to what is written."""
    grads = tensors([(i * 37 % 5000 + 1,) for i in range(700)], "mixed")
    want, clipped = O.clip(doubles(grads), 3.0, 1.0)
    norm = gpu.clip_grads(grads, 3.0)
    assert abs(norm.item() - want) <= 2 * O.STEP * want
    for a, b in zip(grads, clipped):
        close(a, b, a.dtype)


def test_same_bits_every_time(gpu):
    grads = tensors([(1000, 999), (31,), (50_000,)], "mixed")
    assert len({gpu.grad_norm(grads).item() for _ in range(10)}) == 1
    outs = []
    for _ in range(5):
        out = [torch.empty_like(g) for g in grads]
        gpu.clip_grads(grads, 1.0, out=out)
        outs.append(out)
    assert all(torch.equal(a, b) for out in outs for a, b in zip(out, outs[0]))


def test_more_than_31_bits_of_elements(gpu):
    g = torch.ones((1 << 31) + 12_345, device="cuda", dtype=torch.bfloat16)
    g[-1] = 3.0
    want = math.sqrt(g.numel() + 8)
    norm = gpu.clip_grads([g], want / 2)
    assert abs(norm.item() - want) <= 2 * O.STEP * want
    assert (g[:-1].view(-1)[:: 1 << 20] == 0.5).all() and (g[-12_400:-1] == 0.5).all() and g[-1] == 1.5


def test_recorded_and_replayed(gpu):
    shapes = [(300, 400), (7,), (90_000,)] + [(50,)] * 130
    grads = tensors(shapes, "mixed")
    out = [torch.empty_like(g, dtype=torch.float32) for g in grads]
    gpu.clip_grads(grads, 1.0, out=out)
    graphs, norms = [], []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, pool=graphs[0].pool() if graphs else None):
            norms.append(gpu.clip_grads(grads, 1.0, out=out))
        graphs.append(graph)
    for turn in range(4):
        for g in grads:
            g.normal_()
        want = [torch.empty_like(o) for o in out]
        norm = gpu.clip_grads(grads, 1.0, out=want)
        for graph, n in zip(graphs, norms):
            for o in out:
                o.fill_(9.0)
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(n, norm) and all(torch.equal(a, b) for a, b in zip(out, want)), turn


def test_gradients_of_a_step(gpu):
    """After backward(), in the parameters' own gradients, on a stream of its own."""
    table = torch.randn(50, 16, device="cuda", requires_grad=True)
    out = torch.randn(50, 16, device="cuda", requires_grad=True)
    rows = gpu.embed(table, torch.arange(20, device="cuda"))
    gpu.token_logprobs(rows @ out.t(), torch.arange(20, device="cuda"))[0].sum().backward()
    want, clipped = O.clip(doubles([table.grad, out.grad]), 0.5, 1.0)
    version = table.grad._version
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        norm = gpu.clip_grads([p.grad for p in (table, out)], 0.5)
    torch.cuda.current_stream().wait_stream(side)
    assert abs(norm.item() - want) <= 2 * O.STEP * want and table.grad._version > version
    for p, b in zip((table, out), clipped):
        close(p.grad, b, torch.float32)


def test_refusals(gpu):
    g = torch.ones(10, 10, device="cuda")
    for bad, error in [
        (lambda: gpu.grad_norm([g.cpu()]), TypeError), (lambda: gpu.grad_norm([g.double()]), TypeError), (lambda: gpu.grad_norm([g.int()]), TypeError),
        (lambda: gpu.grad_norm([g[:, :5]]), ValueError), (lambda: gpu.grad_norm([g[:1].expand(3, 10)]), ValueError), (lambda: gpu.grad_norm([g], float("nan")), ValueError),
        (lambda: gpu.grad_norm([g.clone().requires_grad_()]), ValueError), (lambda: gpu.clip_grads([g], -1.0), ValueError), (lambda: gpu.clip_grads([g], float("nan")), ValueError),
        (lambda: gpu.clip_grads([g], 1.0, float("inf")), ValueError), (lambda: gpu.clip_grads([g, g], 1.0), ValueError), (lambda: gpu.clip_grads([g[:6], g[5:]], 1.0), ValueError),
        (lambda: gpu.clip_grads([g], 1.0, out=[]), ValueError), (lambda: gpu.clip_grads([g], 1.0, out=[g.half()]), TypeError),
        (lambda: gpu.clip_grads([g], 1.0, out=[g.t().contiguous().t()]), ValueError), (lambda: gpu.clip_grads([g], 1.0, out=[g[:5]]), ValueError),
        (lambda: gpu.clip_grads([g[:5], g[5:]], 1.0, out=[g[5:], g[:5]]), ValueError), (lambda: gpu.clip_grads([g[:5]], 1.0, out=[g[1:6]]), ValueError),
        (lambda: gpu.clip_grads([g.clone().requires_grad_()], 1.0), ValueError), (lambda: gpu.clip_grads([g], 1.0, out=[g.clone().requires_grad_()]), ValueError),
    ]:
        before = g.clone()
        with pytest.raises(error):
            bad()
        assert torch.equal(g, before)
    with torch.no_grad():
        p = g.clone().requires_grad_()
        gpu.clip_grads([p], 1.0)
        assert abs(p.norm().item() - 1.0) < 1e-5
