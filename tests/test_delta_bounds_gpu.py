"""The ends of the gated delta rule's buffers: sequences whose last chunk has one, two, three or 61
tokens, value heads that fill no tile. Operands are slices of larger buffers that hold NaN behind the
last token, outputs and workspaces lie between guard values; neither may be touched. Results are those
of dense operands, to the bit, and the oracle's within the parity tests' tolerances (four fp32 sums of
at most 192 terms: 5e-5 of the terms' size; bf16's half step 2^-8 besides)."""
import ctypes

import pytest
import torch
import torch.nn.functional as F

from oracle import delta_oracle as O

pytestmark = pytest.mark.gpu
DEV = "cuda"
F32, BF16 = 5e-5, 2.0 ** -8 + 1e-4
NAMES = ("q", "k", "v", "g", "beta")
TYPES = pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
# the last one has 256 heads of two 32-column tiles: a workgroup of a pass takes 32 columns there (bf16)
SHAPES = pytest.mark.parametrize("shape", [(2, 65, 1, 1, 24, 8), (2, 130, 2, 6, 40, 24), (3, 67, 1, 2, 64, 40), (2, 189, 2, 2, 72, 40),
                                           (2, 1, 1, 3, 16, 24), (4, 66, 64, 64, 16, 40)], ids=lambda s: "x".join(map(str, s)))


class Dims(ctypes.Structure):
    _fields_ = [(n, ctypes.c_int) for n in ("B", "T", "Hk", "H", "K", "V")]


class Rows(ctypes.Structure):
    _fields_ = [("p", ctypes.c_void_p), ("sb", ctypes.c_int64), ("st", ctypes.c_int64), ("sh", ctypes.c_int64)]


def _inputs(B, T, Hk, H, K, V, dtype):
    gen = torch.Generator().manual_seed(31 * T + K + V)

    def normal(*s):
        return torch.randn(*s, generator=gen)

    q, k = (F.normalize(F.silu(normal(B, T, Hk, K)), dim=-1) for _ in range(2))
    x = [q, k, normal(B, T, H, V), -0.3 * F.softplus(normal(B, T, H)), torch.sigmoid(normal(B, T, H))]
    return [t.to(dtype) for t in x], normal(B, T, H, V).to(dtype), normal(B, H, K, V), normal(B, H, K, V)


def _behind(t, value=float("nan")):
    """t on the GPU as a slice of a buffer with `value` in 64 more tokens of every batch row."""
    buf = torch.full((t.shape[0], t.shape[1] + 64, *t.shape[2:]), value, dtype=t.dtype, device=DEV)
    buf[:, :t.shape[1]] = t.to(DEV)
    return buf[:, :t.shape[1]]


class Guarded:
    """`count` values of a type between two guards of 16384 values each."""

    def __init__(self, count, dtype):
        self.n, self.pad = count, 16384
        self.buf = torch.full((count + 2 * self.pad,), 77, dtype=dtype, device=DEV)
        self.t = self.buf[self.pad:self.pad + count]

    def untouched(self):
        return bool((self.buf[:self.pad] == 77).all()) and bool((self.buf[self.pad + self.n:] == 77).all())


def _off(a, b):
    b = b.detach().double().cpu()
    return float((a.detach().double().cpu() - b).norm() / b.norm().clamp_min(1e-30))


@TYPES
@SHAPES
def test_guards(shape, dtype):
    from gruboros_amd import _lib

    L = _lib.lib()
    B, T, Hk, H, K, V = shape
    xs, do, h0, ds = _inputs(*shape, dtype)
    dev, dod, h0d, dsd = [_behind(t) for t in xs], _behind(do), h0.to(DEV), ds.to(DEV)
    code, d, stream = int(dtype == torch.bfloat16), Dims(*shape), torch.cuda.current_stream().cuda_stream

    def ref(x):
        return ctypes.cast(ctypes.pointer(x), ctypes.c_void_p)

    def rows(t):
        s = t.stride()
        return ref(Rows(t.data_ptr(), s[0], s[1], s[2]))

    ops = [rows(t) for t in dev]
    kept_bytes, ws_bytes = L.mg_delta_fwd_workspace_bytes(code, ref(d), 1), L.mg_delta_bwd_workspace_bytes(code, ref(d))
    kept, ws = Guarded(kept_bytes, torch.uint8), Guarded(ws_bytes, torch.uint8)
    o, state = Guarded(B * T * H * V, dtype), Guarded(B * H * K * V, torch.float32)
    grads = [Guarded(t.numel(), dtype) for t in xs] + [Guarded(h0.numel(), torch.float32)]
    scale = ctypes.c_float(K ** -0.5)
    _lib.check(L.mg_delta_fwd(code, ref(d), *ops, scale, h0d.data_ptr(), o.t.data_ptr(), state.t.data_ptr(), 1, kept.t.data_ptr(),
                              kept_bytes, stream))
    torch.cuda.synchronize()
    assert all(g.untouched() for g in (o, state, kept))
    _lib.check(L.mg_delta_bwd(code, ref(d), *ops, scale, kept.t.data_ptr(), kept_bytes, rows(dod), dsd.data_ptr(),
                              *(g.t.data_ptr() for g in grads), ws.t.data_ptr(), ws_bytes, stream))
    torch.cuda.synchronize()
    assert all(g.untouched() for g in (kept, ws, *grads))

    rs = [t.double().requires_grad_(True) for t in (*xs, h0)]
    ro, rstate = O.gated_delta_rule(*rs)
    want = torch.autograd.grad([ro, rstate], rs, [do.double(), ds.double()])
    tol = F32 if dtype == torch.float32 else BF16
    assert _off(o.t.view(ro.shape), ro) <= tol and _off(state.t.view(rstate.shape), rstate) <= F32
    for n, g, w in zip((*NAMES, "h0"), grads, want):
        if n != "g":
            assert _off(g.t.view(w.shape), w) <= (F32 if n == "h0" else tol), n
        else:
            assert bool(g.t.isfinite().all())


@TYPES
@SHAPES
def test_nan_behind_the_last_token(shape, dtype):
    from gruboros_amd.delta import gated_delta_rule

    xs, do, h0, ds = _inputs(*shape, dtype)

    def run(place):
        leaves = [place(t).requires_grad_(True) for t in xs] + [h0.to(DEV).requires_grad_(True)]
        o, s = gated_delta_rule(*leaves[:5], initial_state=leaves[5], return_state=True)
        return [o, s, *torch.autograd.grad([o, s], leaves, [place(do), ds.to(DEV)])]

    for a, b in zip(run(_behind), run(lambda t: t.to(DEV))):
        assert bool(a.isfinite().all()) and torch.equal(a, b)


@TYPES
def test_broadcast_over_the_tokens(dtype):
    """v and do of one token for all: a distance of zero between rows, where those behind the last
    one are the same memory as those before it."""
    from gruboros_amd.delta import gated_delta_rule

    xs, do, h0, _ = _inputs(2, 130, 2, 6, 40, 24, dtype)
    xs, do, h0 = [t.to(DEV) for t in xs], do[:, :1].to(DEV).expand(-1, 130, -1, -1), h0.to(DEV)
    xs[2] = xs[2][:, :1].expand(-1, 130, -1, -1)

    def run(place):
        leaves = [place(t).detach().requires_grad_(True) for t in xs]
        o = gated_delta_rule(*leaves, initial_state=h0)
        return [o, *torch.autograd.grad(o, leaves, place(do))]

    for a, b in zip(run(lambda t: t), run(lambda t: t.contiguous())):
        assert bool(a.isfinite().all()) and torch.equal(a, b)
