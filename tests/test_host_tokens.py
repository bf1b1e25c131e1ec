"""What the token operators refuse before they touch a GPU: through the C entry points and in Python."""
import ctypes

import pytest
import torch

A = 1 << 20          # an address that is never followed: every call below is refused


def test_entry_points_refuse(oracle):
    from dciknn_cuda_amd import _capi
    lib = _capi.lib()
    inval = -1
    embed = lambda table=A, dtype=0, rows=5, dim=8, stride=8, ids=A, width=8, n=3, out=A: lib.dcih_embed(   # noqa: E731
        table, dtype, rows, dim, stride, ids, width, n, 1.0, out, None)
    for bad in (dict(table=None), dict(dtype=3), dict(dtype=-1), dict(rows=0), dict(rows=1 << 31), dict(dim=0), dict(stride=7), dict(ids=None),
                dict(width=2), dict(n=-1), dict(n=1 << 31), dict(out=None), dict(ids=A + 4), dict(table=A + 2)):
        assert embed(**bad) == inval, bad
        assert lib.dcih_last_error().startswith(b"dcih_embed: ")
    assert embed(n=0, ids=None, out=None) == 0
    need = lib.dcih_embed_grad_work(100, 8, 5)
    assert need > 0 and lib.dcih_embed_grad_work(-1, 8, 5) == inval and lib.dcih_embed_grad_work(1, 0, 5) == inval
    assert lib.dcih_embed_grad_work(1, 8, 0) == inval
    grad = lambda g=A, dtype=0, n=100, dim=8, stride=8, ids=A, width=8, rows=5, out=A, kind=0, work=A, size=need: lib.dcih_embed_grad(   # noqa: E731
        g, dtype, n, dim, stride, ids, width, rows, 1.0, 0, out, kind, work, size, None)
    for bad in (dict(g=None), dict(dtype=4), dict(n=-1), dict(dim=0), dict(stride=1), dict(ids=None), dict(width=1), dict(rows=0), dict(out=None),
                dict(kind=1), dict(dtype=1, kind=2), dict(work=None), dict(size=need - 1), dict(work=A + 8)):
        assert grad(**bad) == inval, bad
    need = lib.dcih_logits_work(4, 90000, 2, 5)
    assert need >= 64
    for bad in ((-1, 9, 0, 0), (4, 0, 0, 0), (4, (1 << 28) + 1, 0, 0), (4, 9, 3, 0), (4, 9, 0, 65), (4, 9, 0, -1)):
        assert lib.dcih_logits_work(*bad) == inval, bad
    logp = lambda z=A, dtype=2, n=4, v=90000, stride=90000, t=A, width=8, temp=1.0, top=5, lp=A, h=A, ids=A, lps=A, stats=None, work=A, size=need: (   # noqa: E731
        lib.dcih_token_logprobs(z, dtype, n, v, stride, t, width, temp, top, lp, h, ids, lps, stats, work, size, None))
    nan, inf = float("nan"), float("inf")
    for bad in (dict(z=None), dict(z=A + 1), dict(dtype=7), dict(n=-1), dict(v=0), dict(stride=89999), dict(t=None), dict(width=3), dict(temp=0.0),
                dict(temp=-1.0), dict(temp=nan), dict(temp=inf), dict(top=65), dict(top=-1), dict(lp=None), dict(h=None), dict(ids=None), dict(lps=None),
                dict(stats=A + 4), dict(work=None), dict(size=need // 2)):
        assert logp(**bad) == inval, bad
    assert logp(v=4, stride=4) == inval                       # five alternatives of four
    assert all(logp(**bad) == inval for bad in (dict(lp=A + 2), dict(h=A + 1), dict(ids=A + 2), dict(lps=A + 3)))
    back = lambda z=A, n=4, v=9, stride=9, t=A, stats=A, grad=1 << 24, gs=9: lib.dcih_token_logprobs_grad(   # noqa: E731
        z, 0, n, v, stride, t, 8, 1.0, stats, None, None, grad, gs, None)
    for bad in (dict(z=None), dict(t=None), dict(stats=None), dict(stats=A + 4), dict(grad=None), dict(gs=8), dict(grad=A + 4), dict(grad=A, gs=12)):
        assert back(**bad) == inval, bad
    distill = lambda z=A, n=4, v=9, ids=A, width=8, t=A, kind=0, k=3, temp=1.0, loss=A, stats=None, grad=None, gs=9, work=A, size=1 << 20: (   # noqa: E731
        lib.dcih_distill(z, 0, n, v, 9, ids, width, t, kind, k, temp, loss, stats, None, grad, gs, work, size, None))
    for bad in (dict(z=None), dict(v=10), dict(ids=None), dict(width=0), dict(t=None), dict(kind=5), dict(k=0), dict(k=1025), dict(temp=0.0), dict(loss=None),
                dict(loss=A + 2), dict(stats=A + 8), dict(grad=A + 4), dict(grad=1 << 24, gs=8), dict(grad=1 << 24, size=63), dict(grad=1 << 24, work=None)):
        assert distill(**bad) == inval, bad
    assert lib.dcih_distill_grad(A, 0, 4, 9, 9, A, 8, A, 0, 3, 1.0, None, None, 1 << 24, 9, None) == inval
    assert lib.dcih_distill_grad(A, 0, 4, 9, 9, A, 8, A, 0, 0, 1.0, A, None, 1 << 24, 9, None) == inval
    assert logp(n=0, t=None, lp=None) == 0 and distill(n=0, ids=None) == 0 and back(n=0, stats=None) == 0


def test_tensors_off_the_gpu_are_refused():
    import dciknn_cuda_amd as D
    z, t = torch.randn(4, 9), torch.zeros(4, dtype=torch.int64)
    ids, teacher = torch.zeros(4, 3, dtype=torch.int64), torch.zeros(4, 3)
    for call in (lambda: D.embed(z, t), lambda: D.embed_grad(z, t, 5), lambda: D.token_logprobs(z, t), lambda: D.distill_loss(z, ids, teacher),
                 lambda: D.distill_step(z, ids, teacher)):
        with pytest.raises(TypeError, match="cuda tensor"):
            call()
    with pytest.raises(TypeError):
        D.embed([[1.0]], t)


def test_workspace_grows_with_what_is_split():
    from dciknn_cuda_amd import _capi
    lib = _capi.lib()
    assert lib.dcih_logits_work(8192, 32000, 2, 20) == 8192 * 16           # rows enough: one workgroup each
    one = lib.dcih_logits_work(1, 131072, 2, 20)
    assert one > 16 and lib.dcih_logits_work(1, 131072, 2, 0) < one
    assert ctypes.sizeof(ctypes.c_int64) == 8 and lib.dcih_logits_work(0, 9, 0, 0) == 0


def test_rows_too_far_apart(oracle):
    """Distances whose product with the number of rows leaves 63 bits."""
    from dciknn_cuda_amd import _capi
    lib, far = _capi.lib(), 1 << 61
    assert lib.dcih_embed(A, 0, 5, 8, far, A, 8, 3, 1.0, A, None) == -1
    assert lib.dcih_embed_grad(A, 0, 3, 8, far, A, 8, 5, 1.0, 0, A, 0, A, 1 << 20, None) == -1
    assert lib.dcih_token_logprobs(A, 0, 4, 9, far, A, 8, 1.0, 0, A, A, None, None, None, A, 1 << 20, None) == -1
    assert lib.dcih_distill(A, 0, 4, 9, 9, A, 8, A, 0, 3, 1.0, A, None, None, 1 << 24, far, A, 1 << 20, None) == -1
