"""Argument errors of the norms around a block: found before anything is enqueued, so they need no GPU."""
import pytest
import torch

from gruboros_amd import _lib

F32, BF16 = 0, 1
ARG, DTYPE, WORKSPACE = 1, 2, 3


def _fwd(L, **kw):
    a = dict(x=4096, ft=BF16, f=4096, g=4096, act=2, wf=4096, scale=None, w=4096, xn=4096, yt=BF16, y=4096, rf=None, rx=None, N=5, D=64,
             eps=1e-6, stream=None)
    a.update(kw)
    return L.mg_block_norm_fwd(*a.values())


def _bwd(L, **kw):
    a = dict(xn=4096, ft=BF16, f=4096, g=4096, act=2, wf=4096, scale=None, w=4096, rf=4096, rx=4096, yt=BF16, dy=4096, dres=None, dx=4096,
             df=4096, dg=4096, dwf=4096, dscale=None, dw=4096, N=5, D=64, ws=4096, wsb=1 << 24, stream=None)
    a.update(kw)
    return L.mg_block_norm_bwd(*a.values())


# (every call below fails its checks before any launch)
def test_forward():
    L = _lib.lib()
    for kw in (dict(N=0), dict(D=0), dict(D=16385), dict(act=3), dict(act=-1), dict(x=None), dict(x=4098), dict(f=None), dict(f=4097),
               dict(g=None), dict(wf=None), dict(w=4098), dict(scale=4098), dict(xn=None), dict(y=None), dict(rf=4096, rx=None),
               dict(ft=F32, f=4098)):
        assert _fwd(L, **kw) == ARG, kw
    assert _fwd(L, ft=2) == DTYPE and _fwd(L, yt=5) == DTYPE


def test_backward():
    L = _lib.lib()
    for kw in (dict(N=0), dict(D=16385), dict(act=7), dict(xn=None), dict(f=None), dict(g=None), dict(rf=None), dict(rx=None), dict(dy=None),
               dict(dres=4098), dict(dx=4098), dict(df=4097), dict(dg=4097), dict(dw=4098), dict(dwf=2), dict(dscale=2), dict(act=0)):
        assert _bwd(L, **kw) == ARG, kw
    assert _bwd(L, ft=2) == DTYPE and _bwd(L, yt=5) == DTYPE
    for kw in (dict(wsb=8), dict(ws=None), dict(ws=4100)):
        assert _bwd(L, **kw) == WORKSPACE, kw
    assert L.mg_block_norm_bwd_workspace_bytes(5, 64) == 2 * 2 * 64 * 4
    assert L.mg_block_norm_bwd_workspace_bytes(0, 64) == 0


def test_cpu_tensors_are_refused():
    from gruboros_amd.norm import add_gated_rms_norm

    x, w = torch.zeros(2, 4), torch.ones(4)
    with pytest.raises(_lib.MingruHipError):
        add_gated_rms_norm(x, x, w, w)
