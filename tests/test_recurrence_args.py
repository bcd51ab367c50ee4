"""Argument errors of the gated linear recurrence: found before anything is enqueued, so they need no GPU."""
import ctypes

import pytest
import torch

from gruboros_amd import _lib

F32, BF16 = 0, 1
ARG, DTYPE, WORKSPACE = 1, 2, 3


class Seq(ctypes.Structure):
    _fields_ = [("p", ctypes.c_void_p), ("sb", ctypes.c_int64), ("st", ctypes.c_int64)]


@pytest.fixture(scope="module")
def L():
    return _lib.lib()


def _seq(p=4096, sb=640, st=64):
    return ctypes.cast(ctypes.pointer(Seq(p, sb, st)), ctypes.c_void_p)


def _fwd(L, **kw):
    a = dict(dtype=BF16, x=_seq(), gi=_seq(), gr=_seq(), decay=4096, c=8.0, h0=None, reset=None, h=4096, last=None, keep=None, B=2, T=300,
             D=64, ws=4096, wsb=1 << 30, stream=None)
    a.update(kw)
    return L.mg_recurrence_fwd(*a.values())


def _bwd(L, **kw):
    a = dict(dtype=BF16, x=_seq(), gi=_seq(), gr=_seq(), decay=4096, c=8.0, h0=None, reset=None, keep=4096, dh=_seq(), dlast=None, dx=4096,
             di=4096, dr=4096, dd=None, dh0=None, B=2, T=300, D=64, ws=4096, wsb=1 << 30, stream=None)
    a.update(kw)
    return L.mg_recurrence_bwd(*a.values())


def _step(L, **kw):
    a = dict(dtype=BF16, x=4096, xl=64, gi=4096, gil=64, gr=4096, grl=64, decay=4096, c=8.0, state=4096, h=4096, B=2, D=64, stream=None)
    a.update(kw)
    return L.mg_recurrence_step(*a.values())


# (every call below fails its checks before any launch)
@pytest.mark.parametrize("call", [_fwd, _bwd], ids=["fwd", "bwd"])
def test_sequences(L, call):
    for kw in (dict(B=0), dict(T=0), dict(D=0), dict(c=-1.0), dict(c=float("nan")), dict(c=float("inf")), dict(x=_seq(p=None)),
               dict(x=_seq(p=4097)), dict(gi=_seq(st=-1)), dict(gr=_seq(sb=-5)), dict(x=_seq(st=1 << 28)), dict(gr=None), dict(decay=None),
               dict(decay=4098), dict(B=1 << 20, D=1 << 12), dict(B=1 << 12, T=1 << 20, D=64)):
        assert call(L, **kw) == ARG, kw
    assert call(L, dtype=2) == DTYPE
    for kw in (dict(wsb=8), dict(ws=None), dict(ws=4100)):
        assert call(L, **kw) == WORKSPACE, kw
        assert b"workspace" in L.mg_last_error()


def test_backward(L):
    for kw in (dict(keep=None), dict(dh=None), dict(dx=None), dict(di=None), dict(dr=None), dict(dlast=4098), dict(dd=4098), dict(dh0=2)):
        assert _bwd(L, **kw) == ARG, kw


def test_step(L):
    for kw in (dict(B=0), dict(D=0), dict(x=None), dict(x=4097), dict(xl=-1), dict(state=None), dict(state=4098), dict(h=None), dict(c=-1.0),
               dict(decay=None), dict(dtype=F32, h=4098)):
        assert _step(L, **kw) == ARG, kw
    assert _step(L, dtype=3) == DTYPE


def test_sizes(L):
    # one tile each way needs no words; else a ticket per chain and eight bytes per tile and channel
    assert L.mg_recurrence_fwd_workspace_bytes(2, 128, 64) == 0
    assert L.mg_recurrence_fwd_workspace_bytes(2, 129, 64) == 16 + 2 * 2 * 64 * 8
    assert L.mg_recurrence_bwd_workspace_bytes(2, 65, 64) == 16 + 2 * 2 * 64 * 8 + 2 * 2 * 64 * 4
    assert L.mg_recurrence_fwd_workspace_bytes(0, 128, 64) == 0
    assert L.mg_recurrence_keep_elems(2, 23, 5) == 2 * 2 * 5


def test_cpu_tensors_are_refused():
    from gruboros_amd.recurrence import gated_recurrence, gated_recurrence_step

    x = torch.zeros(1, 2, 4)
    with pytest.raises(_lib.MingruHipError):
        gated_recurrence(x, x, x, torch.zeros(4))
    with pytest.raises(_lib.MingruHipError):
        gated_recurrence_step(x[:, 0], x[:, 0], x[:, 0], torch.zeros(4), torch.zeros(1, 4))
