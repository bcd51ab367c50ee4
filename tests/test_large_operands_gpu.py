"""The kernels that operands or results beyond the caches take (past 256 MB of the recurrence's operands, 192 MB of the
embedding's results), against float64.

Tolerances before any run. Recurrence: as its other tests, 2e-5 and bfloat16's half step; a state that forgets at
least 0.001 of itself per token of an open gate holds on to the 2100 tokens that they allow for, however long the row.
Its decay's gradient is a sum over 32762 tokens of terms of both signs: 4e-5 of the size that the terms add up to as a
root, as there. Embedding: a value passes 16 sums of its piece, at most 16 pieces, or a quarter of an id's, and the 15
places on either side, then one join of four shares and the scale: (52 + max(16, n / 64)) 2^-24 of the sum of the
sizes for n tokens of an id, and half a step of the table's type. The lookup: the product's half step and the output's.
"""
import pytest
import torch

from oracle.recurrence_oracle import gated_recurrence as oracle

pytestmark = pytest.mark.gpu
DEV = "cuda"
f32, bf16 = torch.float32, torch.bfloat16
HALF = {f32: 2.0 ** -24, bf16: 2.0 ** -8}
TYPES = pytest.mark.parametrize("dtype", [f32, bf16], ids=["f32", "bf16"])


@pytest.fixture(autouse=True)
def _memory():
    yield
    torch.cuda.empty_cache()


def _rel(a, b):
    a, b = a.detach().double().cpu(), b.detach().double().cpu()
    return float((a - b).norm() / b.norm())


@TYPES
@pytest.mark.parametrize("packed", [False, True], ids=["whole", "packed"])
def test_recurrence(packed, dtype):
    """402 MB of x and gates, 537 with the gradient: some channels of every workgroup's first and last columns."""
    from gruboros_amd.recurrence import gated_recurrence

    B, T, D = (2, 16381, 2048) if dtype == bf16 else (1, 16381, 2048)
    tol = 2e-5 + (2.0 ** -8 if dtype == bf16 else 0.0)
    gen = torch.Generator(device=DEV).manual_seed(3)
    n = lambda *s: torch.randn(*s, generator=gen, device=DEV)  # noqa: E731
    rate = -torch.log(0.9 + 0.099 * torch.rand(D, generator=gen, device=DEV)) / 8.0
    leaves = [n(B, T, D).to(dtype), n(B, T, D).to(dtype), n(B, T, D).to(dtype), torch.log(torch.expm1(rate)), n(B, D)]
    dh, dlast = n(B, T, D).to(dtype), n(B, D)
    assert 3 * leaves[0].numel() * leaves[0].element_size() > 1 << 28
    reset = torch.rand(B, T, generator=gen, device=DEV) < 0.002 if packed else None
    for t in leaves:
        t.requires_grad_(True)
    h, last = gated_recurrence(*leaves, reset=reset, return_state=True)
    grads = torch.autograd.grad([h, last], leaves, [dh, dlast])

    at = torch.tensor([0, 3, 63, 64, 1000, 1023, 1984, 2047], device=DEV)
    few = [t.detach()[..., at].double().cpu().requires_grad_(True) for t in leaves]
    want, want_last = oracle(*few, reset=None if reset is None else reset.cpu())
    ref = torch.autograd.grad([want, want_last], few, [dh[..., at].double().cpu(), dlast[..., at].double().cpu()])
    assert _rel(h[..., at], want) <= tol and _rel(last[..., at], want_last) <= 2e-5
    for name, g, r in zip(("x", "input_gate", "decay_gate"), grads, ref):
        assert _rel(g[..., at], r) <= tol, name
    assert _rel(grads[4][..., at], ref[4]) <= 2e-5
    err = (grads[3][at].double().cpu() - ref[3]).norm()
    assert float(err) <= 4e-5 * float(ref[3].norm()) * (B * T) ** 0.5 / 8


def _ids(N, V, gen):
    """Ids of one, few, many and very many tokens, and rows that none has."""
    u = torch.rand(N, generator=gen, dtype=torch.float64)
    ids = (u ** 6 * V).long()  # (the first ids are most)
    ids[torch.rand(N, generator=gen) < 0.2] = V - 1
    ids[torch.rand(N, generator=gen) < 0.01] = V // 2
    return ids


@TYPES
def test_embedding_gradient(dtype):
    from gruboros_amd.embed import scaled_embedding

    V, D, N, scale = (131071 if dtype == bf16 else 50001), 1024, 20000, 1.7
    gen = torch.Generator().manual_seed(1)
    ids = _ids(N, V, gen).to(DEV)
    dy = torch.randn(N, D, generator=gen).to(DEV).to(bf16)
    w = torch.zeros(V, D, dtype=dtype, device=DEV, requires_grad=True)
    assert w.numel() * w.element_size() > 192 << 20
    (g,) = torch.autograd.grad(scaled_embedding(ids, w, scale, bf16), w, dy)
    count = torch.bincount(ids, minlength=V)
    assert int(count.max()) > 16 * 18 and int((count == 0).sum()) > V // 2 and int((count == 1).sum()) > 100
    assert bool((g[count == 0] == 0).all())
    rows = count.nonzero().flatten()
    place = torch.zeros(V, dtype=torch.int64, device=DEV)
    place[rows] = torch.arange(len(rows), device=DEV)
    values = dy.double() * scale
    want = torch.zeros(len(rows), D, dtype=torch.float64, device=DEV).index_add_(0, place[ids], values)
    size = torch.zeros_like(want).index_add_(0, place[ids], values.abs())
    steps = 52 + (count[rows].double() / 64).clamp_min(16)
    lim = steps.unsqueeze(-1) * 2.0 ** -24 * size + HALF[dtype] * want.abs() + 1e-37
    assert bool(((g[rows].double() - want).abs() <= lim).all())


@TYPES
def test_embedding_lookup(dtype):
    from gruboros_amd.embed import scaled_embedding

    V, D = 3000, 1024
    N = 98501 if dtype == bf16 else 49301
    gen = torch.Generator().manual_seed(2)
    ids = torch.randint(-1, V + 1, (N,), generator=gen).to(DEV)
    for table in (f32, bf16):
        w = torch.randn(V, D, generator=gen).to(DEV).to(table)
        y = scaled_embedding(ids, w, 1.7, dtype)
        assert y.numel() * y.element_size() > 192 << 20
        inside = (ids >= 0) & (ids < V)
        assert bool(y[~inside].isnan().all())
        want = w.double()[ids.clamp(0, V - 1)] * 1.7
        lim = (HALF[dtype] + 2.0 ** -23) * want.abs() + 1e-37  # (1.7 itself is a float32)
        assert bool((((y.double() - want).abs() <= lim) | ~inside.unsqueeze(-1)).all())
