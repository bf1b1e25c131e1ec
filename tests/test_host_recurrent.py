"""What the recurrence, the clipping and the verification refuse before they touch a GPU: through the C entry points and in Python."""
import ctypes

import pytest
import torch

A = 1 << 20          # an address that is never followed: every call below is refused
B = 1 << 24


def test_scan_refuses(oracle):
    from dciknn_cuda_amd import _capi
    lib = _capi.lib()
    need = lib.dcih_scan_work(3, 500, 16, 2, 0)
    assert need > 0 and lib.dcih_scan_states(3, 500, 16, 2) > 0 and lib.dcih_scan_states(0, 0, 16, 2) == 0
    for bad in ((-1, 5, 16, 2, 0), (3, -1, 16, 2, 0), (3, 5, 0, 2, 0), (3, 5, (1 << 20) + 1, 2, 0), (3, 5, 16, 3, 0), (3, 5, 16, 2, -1), (3, 5, 16, 2, 7),
                (1 << 31, 5, 16, 2, 0), (1 << 30, 1 << 30, 16, 2, 0)):
        assert lib.dcih_scan_work(*bad) == -1, bad
        assert lib.dcih_last_error().startswith(b"dcih_scan_work: ")
    scan = lambda x=A, dtype=2, rows=3, length=500, dim=16, xr=8000, xs=16, g=A, gr=8000, gs=16, flags=0, state=None, bounds=None, width=4, packed=0, h=B, last=None, states=None, work=A, size=need: (   # noqa: E731
        lib.dcih_scan(x, dtype, rows, length, dim, xr, xs, g, gr, gs, flags, state, bounds, width, packed, h, last, states, work, size, None))
    bad_scan = [dict(x=None), dict(x=A + 1), dict(dtype=5), dict(rows=-1), dict(length=1 << 31), dict(dim=0), dict(xr=-1), dict(xs=-16), dict(g=None), dict(gr=-1),
                dict(xs=1 << 58), dict(gr=1 << 60), dict(flags=4), dict(state=A + 2), dict(bounds=A + 2), dict(bounds=A, width=3), dict(packed=2), dict(rows=1, packed=2),
                dict(h=None), dict(h=A), dict(h=A + 100), dict(h=B + 1), dict(last=A + 1), dict(states=A + 3), dict(state=A, last=A + 4), dict(last=B), dict(last=A + 64), dict(work=None), dict(work=A + 8), dict(size=need - 1)]
    for bad in bad_scan:
        assert scan(**bad) == -1, bad
        assert lib.dcih_last_error().startswith(b"dcih_scan: ")
    back = lambda x=A, dtype=2, rows=3, length=500, dim=16, xr=8000, xs=16, g=A, gr=8000, gs=16, flags=0, state=None, bounds=None, width=4, packed=0, states=A, dh=None, dl=None, dx=B, dg=None, ds=None, work=A, size=need: (   # noqa: E731
        lib.dcih_scan_grad(x, dtype, rows, length, dim, xr, xs, g, gr, gs, flags, state, bounds, width, packed, states, dh, dl, dx, dg, ds, work, size, None))
    for bad in [b for b in bad_scan if not set(b) & {"h", "last", "states"}] + [
            dict(states=None), dict(states=A + 2), dict(dx=A), dict(dg=A + 16), dict(dx=B + 1), dict(dh=B + 32), dict(dh=A + 1), dict(dl=A + 2), dict(ds=A + 1)]:
        assert back(**bad) == -1, bad
        assert lib.dcih_last_error().startswith(b"dcih_scan_grad: ")
    # nothing to do
    assert scan(rows=0, x=None, g=None, h=None) == 0 and scan(length=0, x=None, g=None, h=None) == 0 and back(length=0, x=None, g=None, states=None) == 0
    assert back(length=0, flags=2, dg=B) == -1


def test_clip_refuses(oracle):
    from dciknn_cuda_amd import _capi
    lib = _capi.lib()

    def spans(*fields):
        return (_capi.Span * len(fields))(*[_capi.Span(*f) for f in fields])

    good = (A, A, 100, 0, 0)
    need = lib.dcih_clip_work(spans(good), 1)
    assert need >= 16 and lib.dcih_clip_work(None, 0) > 0
    clip = lambda s=(good,), n=None, most=1.0, scale=1.0, norm=A, work=A, size=1 << 20: lib.dcih_clip(spans(*s), len(s) if n is None else n, most, scale, norm, work, size, None)   # noqa: E731
    norm = lambda s=(good,), n=None, scale=1.0, to=A, work=A, size=1 << 20: lib.dcih_grad_norm(spans(*s), len(s) if n is None else n, scale, to, work, size, None)   # noqa: E731
    nan, inf = float("nan"), float("inf")
    for bad in (dict(n=-1), dict(s=((None, A, 1, 0, 0),)), dict(s=((A + 2, A, 1, 0, 0),)), dict(s=((A, A, -1, 0, 0),)), dict(s=((A, A, 1 << 60, 0, 0),)), dict(s=((A, A, 1, 3, 0),)),
                dict(s=((A, A, 1 << 54, 0, 0),)), dict(scale=nan), dict(scale=inf), dict(work=None), dict(work=A + 8), dict(size=8)):
        assert clip(**bad) == -1 and norm(**bad) == -1, bad
        assert lib.dcih_last_error().startswith(b"dcih_grad_norm: ")
    for bad in (dict(s=((A, None, 1, 0, 0),)), dict(s=((A, B, 1, 2, 1),)), dict(s=((A, B, 1, 0, 2),)), dict(s=((A, A + 4, 100, 0, 0),)), dict(s=((A, A, 100, 2, 0),)), dict(s=((A, B + 2, 100, 2, 0),)),
                dict(most=-1.0), dict(most=nan), dict(norm=None), dict(norm=A + 1)):
        assert clip(**bad) == -1, bad
    assert norm(to=None) == -1 and norm(to=A + 2) == -1
    assert ctypes.sizeof(_capi.Span) == 32


def test_verify_refuses(oracle):
    from dciknn_cuda_amd import _capi
    lib = _capi.lib()
    need = lib.dcih_verify_work(4, 3, 9000, 2)
    assert need > 0 and lib.dcih_verify_work(0, 0, 1, 0) == 0
    for bad in ((-1, 3, 9000, 2), (4, -1, 9000, 2), (4, 257, 9000, 2), (4, 3, 0, 2), (4, 3, (1 << 28) + 1, 2), (4, 3, 9000, 4), (1 << 30, 3, 9000, 2)):
        assert lib.dcih_verify_work(*bad) == -1, bad
    nan, inf = float("nan"), float("inf")
    verify = lambda z=A, dtype=2, n=4, k=3, v=9000, stride=9000, ids=A, width=8, u=A, sids=None, swidth=8, t=None, kind=0, slots=5, temp=1.0, tok=A, acc=A, lp=A, work=A, size=need: (   # noqa: E731
        lib.dcih_verify(z, dtype, n, k, v, stride, ids, width, u, sids, swidth, t, kind, slots, temp, tok, acc, lp, work, size, None))
    for bad in (dict(z=None), dict(z=A + 1), dict(dtype=3), dict(n=-1), dict(n=1 << 30), dict(k=-1), dict(k=257), dict(v=0), dict(stride=8999), dict(stride=1 << 60), dict(ids=None),
                dict(ids=A + 4), dict(width=2), dict(u=None), dict(u=A + 2), dict(sids=A), dict(sids=A, t=A, slots=0), dict(sids=A, t=A, slots=1025), dict(sids=A, t=A, kind=3),
                dict(sids=A + 4, t=A), dict(sids=A, t=A + 1), dict(temp=0.0), dict(temp=-1.0), dict(temp=nan), dict(temp=inf), dict(tok=None), dict(tok=A + 1), dict(acc=None), dict(lp=None),
                dict(lp=A + 2), dict(work=None), dict(work=A + 4), dict(size=need - 1)):
        assert verify(**bad) == -1, bad
        assert lib.dcih_last_error().startswith(b"dcih_verify: ")
    assert verify(n=0, ids=None, u=None, tok=None) == 0


def test_tensors_off_the_gpu_are_refused():
    import dciknn_cuda_amd as D
    x, ids = torch.zeros(2, 3, 8), torch.zeros(2, 2, dtype=torch.int64)
    for call in (lambda: D.gated_scan(x, x), lambda: D.grad_norm([x]), lambda: D.clip_grads([x], 1.0), lambda: D.verify_drafts(x, ids, torch.zeros(2, 3))):
        with pytest.raises(TypeError, match="cuda tensor"):
            call()
    with pytest.raises(TypeError):
        D.gated_scan([[1.0]], x)
    with pytest.raises(TypeError):
        D.grad_norm([1.0])
    assert D.grad_norm([]).item() == 0.0 and D.clip_grads(iter(()), 1.0).item() == 0.0


def test_what_a_scan_keeps_grows_with_the_tiles(oracle):
    """The states for the gradient: one of 32 bits a channel for every tile; a workspace for long rows only."""
    from dciknn_cuda_amd import _capi
    lib = _capi.lib()
    one, many = lib.dcih_scan_states(1, 1, 2048, 2), lib.dcih_scan_states(1, 100_000, 2048, 2)
    assert one == 2048 and 2048 * 100_000 / 256 <= many <= 2048 * 100_000 / 64
    assert lib.dcih_scan_states(8, 4096, 2048, 2) == 8 * lib.dcih_scan_states(1, 4096, 2048, 2)
    assert lib.dcih_scan_work(1, 1 << 30, 1, 0, 1) > 0
