"""Arrays that one call writes over others that it reads or writes: refused by the C entry points before they touch a GPU."""
import pytest

X, G, H, S, L, K, W, B = (i << 24 for i in range(1, 9))        # addresses that are never followed: every call below is refused
ROWS, LENGTH, DIM, BF16 = 3, 500, 16, 2
CELLS, STATES = ROWS * LENGTH * DIM * 2, ROWS * DIM * 4


@pytest.fixture(scope="module")
def lib():
    from dciknn_cuda_amd import _capi
    return _capi.lib()


def scan(lib, h=H, state=S, bounds=B, last=L, kept=K, x=X, gates=G, flags=0, packed=0, rows=ROWS, width=4):
    return lib.dcih_scan(x, BF16, rows, LENGTH, DIM, LENGTH * DIM, DIM, gates, LENGTH * DIM, DIM, flags, state, bounds, width, packed, h, last, kept, W, 1 << 30, None)


def scan_grad(lib, dx=H, dg=H + (1 << 22), ds=L, x=X, gates=G, state=S, bounds=B, kept=K, dh=X + (1 << 22), dl=L + (1 << 22), flags=0, length=LENGTH):
    return lib.dcih_scan_grad(x, BF16, ROWS, length, DIM, LENGTH * DIM, DIM, gates, LENGTH * DIM, DIM, flags, state, bounds, 4, 0, kept, dh, dl, dx, dg, ds, W, 1 << 30, None)


SCAN = [dict(h=S), dict(h=S - CELLS + 4), dict(h=S + STATES - 2), dict(h=B), dict(h=B + 4 * ROWS - 2), dict(h=K), dict(kept=X), dict(kept=G + 64), dict(kept=S), dict(kept=B + 8), dict(kept=L),
        dict(last=B), dict(last=B + 4 * ROWS - 4), dict(last=K + 64), dict(kept=H + CELLS - 4), dict(last=L, bounds=L + STATES - 4),
        # offsets: one more than there are sequences
        dict(rows=1, packed=3, h=B + 4 * 4 - 2), dict(rows=1, packed=3, width=8, last=B + 8 * 4 - 4)]


@pytest.mark.parametrize("bad", SCAN, ids=str)
def test_scan(lib, bad):
    assert scan(lib, **bad) == -1
    assert b"overlap" in lib.dcih_last_error()


GRAD = [dict(ds=L + (1 << 22)), dict(ds=S), dict(ds=S + STATES - 4), dict(ds=B + 4), dict(ds=K), dict(ds=X), dict(ds=X + (1 << 22)), dict(ds=G + 32), dict(dx=H, dg=H), dict(dx=H, dg=H + CELLS - 2),
        dict(dx=H, ds=H + 4), dict(dg=L - CELLS + 4), dict(dx=S), dict(dx=K + 64), dict(dx=L + (1 << 22)), dict(dx=B), dict(dg=K), dict(dg=B + 8), dict(dh=H), dict(dl=H + 4),
        # shared gates: a gradient of one row
        dict(flags=2, dg=G), dict(flags=2, dg=X + 2), dict(flags=2, dg=H + CELLS - 2), dict(flags=2, dg=L), dict(flags=2, dg=K + 4), dict(flags=2, dg=S + 4),
        # without tokens the gradient by the states is passed on: not in the place of what it is passed on from
        dict(length=0, ds=L + (1 << 22) + 4)]


@pytest.mark.parametrize("bad", GRAD, ids=str)
def test_scan_grad(lib, bad):
    assert scan_grad(lib, **bad) == -1
    assert b"overlap" in lib.dcih_last_error()


def verify(lib, tokens=H, accepted=K, logprobs=L, drafts=X, uniforms=G, ids=S, teacher=B):
    return lib.dcih_verify(W, BF16, 4, 3, 9000, 9000, drafts, 8, uniforms, ids, 4, teacher, BF16, 5, 1.0, tokens, accepted, logprobs, 9 << 24, 1 << 30, None)


ROW = 4 * 4 * 4           # bytes of what has a number for each row of logits


@pytest.mark.parametrize("bad", [
    dict(tokens=X), dict(tokens=X + 4 * 3 * 8 - 4), dict(tokens=G), dict(tokens=S + 4 * 3 * 5 * 4 - 4), dict(tokens=B), dict(tokens=B + 4 * 3 * 5 * 2 - 4), dict(tokens=L), dict(tokens=K + 12),
    dict(tokens=W + 16 * 9000 * 2 - 4), dict(accepted=X), dict(accepted=G + ROW - 4), dict(accepted=L + 8), dict(accepted=S), dict(accepted=W), dict(logprobs=G + 4), dict(logprobs=X),
    dict(logprobs=S + 16), dict(logprobs=B), dict(logprobs=W + 1000), dict(logprobs=H, tokens=H + ROW - 4), dict(logprobs=G, tokens=G), dict(logprobs=G, accepted=G)], ids=str)
def test_verify(lib, bad):
    assert verify(lib, **bad) == -1
    assert b"overlap" in lib.dcih_last_error()
