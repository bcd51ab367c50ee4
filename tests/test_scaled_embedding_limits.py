"""Rows of the scaled embedding that 32-bit columns do not hold are refused before anything is enqueued: no GPU needed."""
import pytest

from gruboros_amd import _lib

F32, ARG = 0, 1


@pytest.mark.parametrize("D", [1 << 30, (1 << 31) - 1000, (1 << 31) - 1])
def test_widths(D):
    L = _lib.lib()
    assert L.mg_embedding_fwd(8, 4096, 1, F32, 4096, 1, D, 1.0, F32, 4096, None) == ARG
    assert b"D" in L.mg_last_error()
    assert L.mg_embedding_sorted_bwd_workspace_bytes(1, D, 1) == 0
    assert L.mg_embedding_sorted_bwd(8, 4096, 1, F32, 4096, D, 1, 1.0, -1, F32, 4096, 4096, 1 << 62, None) == ARG
    assert L.mg_embedding_sorted_bwd_workspace_bytes(1, (1 << 30) - 1, 1) > 0
