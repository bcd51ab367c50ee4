"""Sizes of the gated delta rule whose launches would have 2^32 threads or more: refused before
anything is enqueued, so the test needs no GPU. The largest that are taken pass the same checks and
are refused for what comes after them."""
import ctypes
import os
import re

import pytest

from gruboros_amd import _lib
from gruboros_amd.build import LIB_PATH


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


def _arg_error():
    text = open(os.path.join(os.path.dirname(LIB_PATH), "..", "include", "mingru_hip.h")).read()
    return int(re.search(r"MG_ERR_ARG\s*=?\s*(-?\d+)", text).group(1))


@pytest.mark.parametrize("B, H, V, good", [(1 << 20, 16, 32, False), (1 << 20, 15, 32, True), (1 << 17, 16, 256, False),
                                           (1 << 17, 15, 256, True), (1 << 22, 1 << 22, 8, False), (5592405, 1, 96, True),
                                           (5592406, 1, 96, False)])
def test_step(L, B, H, V, good):
    d = Dims(B, 1, H, H, 8, V)
    # (no state: the check behind this one)
    rc = L.mg_delta_step(0, _ref(d), 4096, 4096, 4096, 4096, 4096, ctypes.c_float(1.0), None, 4096, None)
    assert rc == _arg_error() and (b"state" if good else b"2^24") in L.mg_last_error()


@pytest.mark.parametrize("B, T, H, V, good", [(1 << 18, 1, 16, 8, False), (1 << 18, 1, 15, 8, True), (1 << 15, 1, 16, 256, False),
                                              (1 << 15, 1, 15, 256, True), (1 << 10, 64 << 10, 8, 8, False),
                                              (1 << 10, 64 << 10, 7, 8, True), (1 << 30, 1 << 30, 4, 8, False)])
def test_sequences(L, B, T, H, V, good):
    d = Dims(B, T, H, H, 8, V)
    for size in (L.mg_delta_fwd_workspace_bytes(0, _ref(d), 1), L.mg_delta_bwd_workspace_bytes(0, _ref(d))):
        assert (size > 0) == good
    none = Rows(None, 0, 0, 0)
    rc = L.mg_delta_fwd(0, _ref(d), *[_ref(none)] * 5, ctypes.c_float(1.0), None, 4096, None, 0, 4096, 1 << 62, None)
    assert rc == _arg_error() and (b"q is NULL" if good else b"2^23") in L.mg_last_error()
    rc = L.mg_delta_bwd(0, _ref(d), *[_ref(none)] * 5, ctypes.c_float(1.0), 4096, 1 << 62, _ref(none), None, *[4096] * 5, None, 4096,
                        1 << 62, None)
    assert rc == _arg_error() and (b"q is NULL" if good else b"2^23") in L.mg_last_error()
