"""What `verify_drafts` draws behind a refused draft where little or nothing is left of a part of its row, and rows without slots."""
import math

import numpy as np
import pytest
import torch

import recurrent_oracles as O
from test_gpu_verify import check

pytestmark = pytest.mark.gpu
CHUNK = 2048             # entries of a row that are added up by one wavefront
BELOW_1 = 1.0 - 2.0 ** -24


def some_live(n, v, live, dtype, seed):
    """Rows [n, 2, v] in which nothing but `live` is possible, of many magnitudes."""
    g = torch.Generator().manual_seed(seed)
    z = torch.full((n, 2, v), -math.inf)
    z[:, :, live] = torch.randn(n, 2, len(live), generator=g) + 10.0 * torch.randn(n, 2, 1, generator=g)
    return z.to(dtype)


def by_slots(drafts, slots=3):
    """The draft for certain, as a distribution: in one slot, the others empty or in vain."""
    ids = torch.full((*drafts.shape, slots), -1)
    ids[:, :, 1], ids[:, :, 2] = drafts, 0
    teacher = torch.zeros(*drafts.shape, slots)
    teacher[:, :, 2] = -math.inf
    return ids, teacher


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("slots", [False, True])
@pytest.mark.parametrize("draft", [5, CHUNK + 700, 3 * CHUNK + 1], ids=["first", "middle", "last"])
def test_draft_alone_in_its_chunk(gpu, draft, slots, dtype):
    """The other possible tokens are in other chunks: of the draft's nothing may be left, with the least and the largest number."""
    others = [t for t in (900, CHUNK + 3, CHUNK + 4, 2 * CHUNK + 9, 4 * CHUNK - 1) if t // CHUNK != draft // CHUNK]
    z = some_live(300, 4 * CHUNK, [draft] + others, dtype, seed=draft)
    drafts = torch.full((300, 1), draft)
    u = torch.full((300, 2), BELOW_1)
    for number in (0.0, 2.0 ** -60, BELOW_1, 1.0):
        u[:, 1] = number
        check(gpu, z, drafts, u, *(by_slots(drafts) if slots else ()), on_border=True)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
def test_slots_that_take_whole_chunks(gpu, dtype):
    """Two of four chunks hold nothing but what the slots take off."""
    live = [7, 8, CHUNK + 1, 2 * CHUNK, 2 * CHUNK + 1, 3 * CHUNK + 5]
    z = some_live(300, 4 * CHUNK, live, dtype, seed=2)
    z[:, :, [7, 8]] -= 4.0
    z[:, :, [2 * CHUNK, 2 * CHUNK + 1]] -= 4.0
    ids = torch.tensor([8, 2 * CHUNK, 7, -1, 2 * CHUNK + 1, 2 * CHUNK]).expand(300, 1, 6).contiguous()
    drafts = torch.full((300, 1), 8)
    teacher = torch.randn(300, 1, 6, generator=torch.Generator().manual_seed(3))
    u = torch.full((300, 2), BELOW_1)
    for number in (0.0, 1.0):
        u[:, 1] = number
        check(gpu, z, drafts, u, ids, teacher, on_border=True)


@pytest.mark.parametrize("live", [[3], [CHUNK + 5], [9, 3 * CHUNK]], ids=str)
@pytest.mark.parametrize("draft", [1, 2 * CHUNK + 1, 4 * CHUNK, 1 << 40])
def test_nothing_left(gpu, live, draft):
    """q is p, and the draft is none of its tokens, or beyond the vocabulary: drawn from p itself."""
    z = some_live(200, 4 * CHUNK, live, torch.float32, seed=4)
    ids = torch.tensor(live + [-1]).expand(200, 1, -1).contiguous()
    teacher = torch.cat([z[:, :1, live], torch.zeros(200, 1, 1)], 2)
    drafts = torch.full((200, 1), draft)
    for number in (0.0, 0.3, 0.5, BELOW_1):
        u = torch.full((200, 2), number)
        check(gpu, z, drafts, u, ids, teacher, on_border=True)


@pytest.mark.parametrize("slots", [False, True])
@pytest.mark.parametrize("draft_chunk", [0, 1, 2])
def test_little_left(gpu, draft_chunk, slots):
    """The draft had all but 1e-7 of its row; random numbers are those of 32 bits next to the borders of what is left.

    Of that 64 bits know all but 1e-15, where the row is known to some 1e-14: by differences of the row's sums a border would be off by 1e-7."""
    g = torch.Generator().manual_seed(5 + draft_chunk)
    n, live = 400, [17, CHUNK + 17, 2 * CHUNK + 17]
    draft = draft_chunk * CHUNK + 1000
    z = torch.full((n, 2, 3 * CHUNK), -math.inf)
    z[:, :, draft] = 30.0 * torch.rand(n, 1, generator=g) - 15.0
    z[:, :, live] = z[:, :, draft, None] - 17.2 + 0.5 * torch.rand(n, 2, 3, generator=g)
    drafts = torch.full((n, 1), draft)
    for border in range(2):
        for way in (0.0, 1.0):
            w = torch.softmax(z[:, 0, live].double(), 1).cumsum(1)[:, border].numpy()
            number = w.astype(np.float32)
            for _ in range(100):
                close = (number - w) * (1 if way else -1) < 1e-9
                number = np.where(close, np.nextafter(number, np.float32(way)), number)
            u = torch.full((n, 2), BELOW_1)
            u[:, 1] = torch.from_numpy(number)
            got = check(gpu, z, drafts, u, *(by_slots(drafts) if slots else ()))
            assert not got[1].any()


@pytest.mark.parametrize("lead", [0.0, 17.0])
def test_large_vocabulary(gpu, lead):
    """More chunks than are added up beside the slots, and than a workgroup has threads; the draft has half of its row, or all but 1e-7."""
    v, draft, others = 1_400_000, 600_001, [600_000 + CHUNK, 1_300_007, 1_399_999]
    z = some_live(6, v, [draft] + others, torch.float32, seed=7)
    z[:, :, draft] = z[:, :, others].logsumexp(2) + lead
    drafts = torch.full((6, 1), draft)
    u = torch.full((6, 2), BELOW_1)
    for number in (0.0, 0.4, 0.9):
        u[:, 1] = number
        check(gpu, z, drafts, u, on_border=True)
        check(gpu, z, drafts, u, *by_slots(drafts), on_border=True)


def test_rows_that_say_nothing_beside_drafts_without_slots(gpu):
    """A draft without filled slots stands where the model holds it for possible: not in a row without probabilities, nor with a number that is none."""
    g = torch.Generator().manual_seed(6)
    z = torch.randn(7, 3, 5000, generator=g)
    drafts = torch.randint(0, 5000, (7, 2), generator=g)
    u = torch.rand(7, 3, generator=g)
    z[0, 0, 4999 - int(drafts[0, 0] == 4999)] = math.nan
    z[1, 1, 77 + int(drafts[1, 1] == 77)] = math.nan
    z[2, 0, 78 + int(drafts[2, 0] == 78)] = math.inf
    z[3, 0] = -math.inf
    u[4, 0], u[5, 1], u[6, 2] = math.nan, math.nan, math.nan
    ids = torch.full((7, 2, 3), -1)
    got = check(gpu, z, drafts, u, ids, torch.randn(7, 2, 3, generator=g), on_border=True)
    assert got[1].tolist() == [0, 1, 0, 0, 0, 1, 2]
    check(gpu, z, drafts, u, ids.clamp(min=5), torch.full((7, 2, 3), -math.inf), on_border=True)
