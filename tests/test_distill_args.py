"""Argument errors of the distillation loss: found before anything is enqueued, so they need no GPU."""
import ctypes

import pytest
import torch

from gruboros_amd import _lib

F32, BF16 = 0, 1
ARG, DTYPE, WORKSPACE = 1, 2, 3


class Seq(ctypes.Structure):
    _fields_ = [("p", ctypes.c_void_p), ("sb", ctypes.c_int64), ("st", ctypes.c_int64)]


def _seq(p=4096, sb=1000, st=100):
    return ctypes.cast(ctypes.pointer(Seq(p, sb, st)), ctypes.c_void_p)


def _call(L, **kw):
    a = dict(zt=BF16, z=_seq(), B=2, T=10, V=100, idb=8, ids=4096, tt=F32, top=4096, K=4, labels=4096, temperature=2.0, alpha=0.5, loss=4096,
             dz=4096, ws=4096, wsb=1 << 20, stream=None)
    a.update(kw)
    return L.mg_distill(*a.values())


# (every call below fails its checks before any launch)
def test_arguments():
    L = _lib.lib()
    for kw in (dict(B=0), dict(T=0), dict(B=1 << 20, T=1 << 20), dict(V=0), dict(V=(1 << 30) + 1), dict(K=0), dict(K=513), dict(z=None),
               dict(z=_seq(p=None)), dict(z=_seq(p=4097)), dict(z=_seq(sb=-1)), dict(z=_seq(st=-1)), dict(ids=None), dict(ids=4100),
               dict(top=None), dict(top=4098), dict(labels=4100), dict(temperature=0.0), dict(temperature=float("nan")), dict(temperature=1e5),
               dict(alpha=-0.1), dict(alpha=1.1), dict(alpha=float("nan")), dict(loss=None), dict(loss=4098), dict(dz=4097)):
        assert _call(L, **kw) == ARG, kw
    for kw in (dict(zt=2), dict(tt=2), dict(idb=2)):
        assert _call(L, **kw) == DTYPE, kw
    for kw in (dict(ws=None), dict(ws=4100), dict(wsb=16)):
        assert _call(L, **kw) == WORKSPACE, kw
    assert L.mg_distill_workspace_bytes(20) == 256 * 2 * 4 + 20 * 2 * 8 and L.mg_distill_workspace_bytes(0) == 0


def test_scale():
    L = _lib.lib()
    for a in ((F32, None, 5, 4096), (F32, 4096, 0, 4096), (F32, 4098, 5, 4096), (BF16, 4097, 5, 4096), (F32, 4096, 5, None)):
        assert L.mg_scale_inplace(*a, None) == ARG, a
    assert L.mg_scale_inplace(2, 4096, 5, 4096, None) == DTYPE


def test_no_capture():
    assert _lib.lib().mg_capture_id(None) == 0


def test_cpu_tensors_are_refused():
    from gruboros_amd.loss import distillation_loss

    with pytest.raises(_lib.MingruHipError):
        distillation_loss(torch.zeros(2, 5), torch.zeros(2, 1, dtype=torch.int64), torch.zeros(2, 1))
