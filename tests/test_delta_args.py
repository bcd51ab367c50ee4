"""Argument errors of the gated delta rule, layer norm and dropout: found before anything is
enqueued, so they need no GPU."""
import ctypes
import os
import re

import pytest
import torch

from gruboros_amd import _lib
from gruboros_amd.build import LIB_PATH

F32, BF16 = 0, 1


class Dims(ctypes.Structure):
    _fields_ = [(n, ctypes.c_int) for n in ("B", "T", "Hk", "H", "K", "V")]


class Rows(ctypes.Structure):
    _fields_ = [("p", ctypes.c_void_p), ("sb", ctypes.c_int64), ("st", ctypes.c_int64), ("sh", ctypes.c_int64)]


@pytest.fixture(scope="module")
def L():
    if not os.path.exists(LIB_PATH):
        pytest.fail(f"{LIB_PATH} not built (run __graft_entry__.build())")
    return _lib.lib()


def _ref(x):
    return ctypes.cast(ctypes.pointer(x), ctypes.c_void_p)


def _codes():
    """(argument, dtype, workspace) error codes as the header has them."""
    text = open(os.path.join(os.path.dirname(LIB_PATH), "..", "include", "mingru_hip.h")).read()
    return tuple(int(re.search(rf"{n}\s*=?\s*(-?\d+)", text).group(1)) for n in ("MG_ERR_ARG", "MG_ERR_DTYPE", "MG_ERR_WORKSPACE"))


GOOD = dict(B=2, T=100, Hk=2, H=4, K=64, V=32)


def _fwd(L, dtype=F32, ptr=4096, st=None, o=4096, ws=4096, ws_bytes=None, **dims):
    d = Dims(**{**GOOD, **dims})
    qk = Rows(ptr, d.T * d.Hk * d.K, d.Hk * d.K if st is None else st, d.K)
    v = Rows(4096, d.T * d.H * d.V, d.H * d.V, d.V)
    g = Rows(4096, d.T * d.H, d.H, 1)
    need = L.mg_delta_fwd_workspace_bytes(dtype, _ref(d), 0)
    return L.mg_delta_fwd(dtype, _ref(d), _ref(qk), _ref(qk), _ref(v), _ref(g), _ref(g), ctypes.c_float(1.0), None, o, None, 0, ws,
                          need if ws_bytes is None else ws_bytes, None)


@pytest.mark.parametrize("dims", [dict(B=0), dict(T=0), dict(H=3), dict(Hk=0), dict(K=4), dict(K=68), dict(K=136), dict(V=260),
                                  dict(V=0), dict(B=1 << 20, T=64 * 1024, H=4), dict(H=1 << 16, Hk=1 << 16, K=8, V=256)],
                         ids=str)
def test_dims(L, dims):
    arg, _, _ = _codes()
    assert _fwd(L, ws_bytes=1 << 60, **dims) == arg


def test_operands(L):
    arg, dtype, workspace = _codes()
    assert _fwd(L, dtype=7) == dtype
    assert _fwd(L, ptr=4104) == arg and b"q" in L.mg_last_error()  # not 16-byte aligned
    assert _fwd(L, ptr=None) == arg
    assert _fwd(L, st=130) == arg  # rows at 8-byte multiples
    assert _fwd(L, st=-128) == arg
    assert _fwd(L, st=1 << 24) == arg  # 64 tokens 4 GiB apart
    assert _fwd(L, o=4104) == arg
    assert _fwd(L, o=None) == arg
    assert _fwd(L, ws=None) == workspace
    assert _fwd(L, ws=4096 + 128) == workspace
    d = Dims(**GOOD)
    assert _fwd(L, ws_bytes=L.mg_delta_fwd_workspace_bytes(F32, _ref(d), 0) - 1) == workspace


def test_backward(L):
    arg, _, workspace = _codes()
    d = Dims(**GOOD)
    qk, v, g = Rows(4096, 12800, 128, 64), Rows(4096, 12800, 128, 32), Rows(4096, 400, 4, 1)
    kept, ws = L.mg_delta_fwd_workspace_bytes(F32, _ref(d), 1), L.mg_delta_bwd_workspace_bytes(F32, _ref(d))
    assert kept > L.mg_delta_fwd_workspace_bytes(F32, _ref(d), 0) > 0 < ws

    def call(dout=v, kept_at=4096, kept_bytes=kept, dq=4096, dbeta=4096, ws_bytes=ws):
        return L.mg_delta_bwd(F32, _ref(d), _ref(qk), _ref(qk), _ref(v), _ref(g), _ref(g), ctypes.c_float(1.0), kept_at, kept_bytes,
                              _ref(dout), None, dq, 4096, 4096, 4096, dbeta, None, 4096, ws_bytes, None)

    assert call(kept_bytes=kept - 1) == workspace
    assert call(kept_at=None) == workspace
    assert call(ws_bytes=ws - 1) == workspace
    assert call(dq=4100) == arg
    assert call(dbeta=None) == arg
    assert call(dout=Rows(4100, 12800, 128, 32)) == arg


def test_step(L):
    arg, dtype, _ = _codes()

    def call(dt=BF16, v=4096, state=4096, **dims):
        d = Dims(**{**GOOD, "T": 1, **dims})
        return L.mg_delta_step(dt, _ref(d), 4096, 4096, v, 4096, 4096, ctypes.c_float(1.0), state, 4096, None)

    assert call(T=2) == arg
    assert call(v=4098) == arg
    assert call(state=4104) == arg
    assert call(state=None) == arg
    assert call(K=12) == arg
    assert call(dt=5) == dtype


def test_layer_norm_and_dropout(L):
    arg, dtype, workspace = _codes()

    def norm(xt=F32, x=4096, delta=None, x_out=None, yt=F32, N=4, D=64, p=0.0, mean=None, rstd=None, seed_p=None):
        return L.mg_layernorm_fwd(xt, x, F32, delta, 4096, None, x_out, yt, 4096, mean, rstd, N, D, ctypes.c_float(1e-5),
                                  ctypes.c_double(p), 0, seed_p, 0, None)

    assert norm(N=0) == norm(D=0) == norm(D=16385) == norm(x=None) == norm(x=4098) == arg
    assert norm(p=1.0) == norm(p=-0.1) == norm(p=float("nan")) == arg
    assert norm(delta=4096) == arg  # no place for the sum
    assert norm(mean=4096) == arg  # without rstd
    assert norm(seed_p=4100) == arg
    assert norm(xt=9) == norm(yt=9) == norm(xt=BF16, delta=4096, x_out=4096) == dtype

    def bwd(ws_bytes):
        return L.mg_layernorm_bwd(F32, 4096, 4096, 4096, 4096, F32, 4096, None, 4096, F32, None, None, None, 4, 64,
                                  ctypes.c_double(0.0), 0, None, 0, 4096, ws_bytes, None)

    need = L.mg_layernorm_bwd_workspace_bytes(4, 64)
    assert need >= 2 * 64 * 4 and bwd(need - 1) == workspace
    assert L.mg_layernorm_bwd_workspace_bytes(4, 16385) == 0

    def drop(xt=F32, x=4096, n=8, p=0.5, residual=None):
        return L.mg_dropout(xt, x, F32, residual, 4096, n, ctypes.c_double(p), 0, None, 0, None)

    assert drop(n=0) == drop(x=4104) == drop(x=None) == drop(p=1.0) == drop(residual=4104) == arg
    assert drop(xt=3) == dtype


def test_cpu_tensors_are_refused():
    from gruboros_amd.delta import gated_delta_rule, gated_delta_step
    from gruboros_amd.dropout import dropout
    from gruboros_amd.norm import add_layer_norm, layer_norm

    x, w = torch.zeros(1, 4, 2, 8), torch.ones(8)
    with pytest.raises(_lib.MingruHipError):
        gated_delta_rule(x, x, x, x[..., 0], x[..., 0])
    with pytest.raises(_lib.MingruHipError):
        gated_delta_step(x[:, 0], x[:, 0], x[:, 0], x[:, 0, :, 0], x[:, 0, :, 0], torch.zeros(1, 2, 8, 8))
    with pytest.raises(_lib.MingruHipError):
        dropout(x, 0.5, 1)
    with pytest.raises(_lib.MingruHipError):
        layer_norm(x, w)
    with pytest.raises(_lib.MingruHipError):
        add_layer_norm(x, x, w)
