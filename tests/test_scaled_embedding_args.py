"""Argument errors of the scaled embedding: found before anything is enqueued, so they need no GPU."""
import pytest
import torch

from gruboros_amd import _lib

F32, BF16 = 0, 1
ARG, DTYPE, WORKSPACE = 1, 2, 3


def _fwd(L, **kw):
    a = dict(idb=8, ids=4096, N=10, wt=F32, w=4096, V=100, D=16, scale=1.0, yt=BF16, y=4096, stream=None)
    a.update(kw)
    return L.mg_embedding_fwd(*a.values())


def _bwd(L, **kw):
    a = dict(idb=8, ids=4096, N=10, gt=BF16, dy=4096, D=16, V=100, scale=1.0, padding=-1, wt=F32, dw=4096, ws=4096, wsb=1 << 30, stream=None)
    a.update(kw)
    return L.mg_embedding_sorted_bwd(*a.values())


# (every call below fails its checks before any launch)
def test_both():
    L = _lib.lib()
    for call in (_fwd, _bwd):
        for kw in (dict(N=0), dict(N=1 << 27), dict(V=0), dict(V=1 << 28), dict(D=0), dict(ids=None), dict(ids=4100)):
            assert call(L, **kw) == ARG, kw
        assert call(L, idb=2) == DTYPE and call(L, wt=2) == DTYPE
    for kw in (dict(w=None), dict(w=4098), dict(y=None), dict(y=4097)):
        assert _fwd(L, **kw) == ARG, kw
    for kw in (dict(dy=None), dict(dy=4097), dict(dw=None), dict(dw=4098)):
        assert _bwd(L, **kw) == ARG, kw
    assert _fwd(L, yt=3) == DTYPE and _bwd(L, gt=3) == DTYPE
    for kw in (dict(ws=None), dict(ws=4112), dict(wsb=100)):
        assert _bwd(L, **kw) == WORKSPACE, kw
    assert L.mg_embedding_sorted_bwd_workspace_bytes(0, 16, 100) == 0
    # a partial row per 32 tokens, and two pairs per token
    assert L.mg_embedding_sorted_bwd_workspace_bytes(6400, 64, 1000) >= 200 * 64 * 4 + 4 * 6400 * 4


def test_cpu_tensors_are_refused():
    from gruboros_amd.embed import scaled_embedding

    with pytest.raises(_lib.MingruHipError):
        scaled_embedding(torch.arange(3), torch.zeros(4, 4))
