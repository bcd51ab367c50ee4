"""Layer norm (with residual add and dropout) and dropout against float64.

Tolerances before any run. float32: a row's sums of n terms are off by at most n 2^-24 of the
terms' size in any order (n <= 16384 would allow 1e-3; trees of lanes and steps of at most 64 +
6 + 16 terms in a row keep them to 86 * 2^-24 = 5e-6), and y, dx pass two of them: 1e-5. dw, db:
sums over rows and workgroups of the same depth: 1e-5. bfloat16: half a step, 2^-8 of each value,
on top: 2^-8 + 1e-5. Dropout: one product and one sum, 2^-23 of each value in fp32, and 2^-8 in bf16.
"""
import numpy as np
import pytest
import torch

from oracle import philox

pytestmark = pytest.mark.gpu
DEV = "cuda"
F32, BF16 = 1e-5, 2.0 ** -8 + 1e-5
f32, bf16 = torch.float32, torch.bfloat16


def _tol(dtype):
    return F32 if dtype == f32 else BF16


def _rel(a, b):
    a, b = a.detach().double().cpu(), b.detach().double().cpu()
    return float((a - b).norm() / b.norm().clamp_min(1e-30))


def _factor(shape, p, seed, offset):
    n = int(np.prod(shape))
    return torch.from_numpy(philox.keep(n, p, seed, offset).astype(np.float64)).view(shape) / (1.0 - p)


def _reference(x, delta, w, b, factor, eps):
    """(xn, y) in float64."""
    if delta is not None:
        x = x + delta * factor
    mu = x.mean(-1, keepdim=True)
    y = (x - mu) / ((x - mu).square().mean(-1, keepdim=True) + eps).sqrt() * w
    return x, (y if b is None else y + b)


@pytest.mark.parametrize("types", [(f32, None, f32), (bf16, None, bf16), (bf16, None, f32), (f32, None, bf16), (f32, bf16, bf16),
                                   (f32, f32, f32), (f32, bf16, f32), (f32, f32, bf16)],
                         ids=lambda t: "-".join("none" if x is None else str(x)[6:] for x in t))
@pytest.mark.parametrize("shape", [(1, 1, 1), (2, 3, 7), (3, 5, 64), (1, 130, 250), (2, 33, 1024), (1, 9, 1001), (2, 5, 2048),
                                   (1, 5, 2050), (1, 3, 5000), (1, 2, 16384), (5000, 1, 24)],
                         ids=lambda s: "x".join(map(str, s)))
def test_layer_norm(shape, types):
    from gruboros_amd.norm import add_layer_norm, layer_norm

    xt, dt, yt = types
    gen = torch.Generator().manual_seed(sum(shape))
    D, p, seed, eps = shape[-1], 0.25, (3 << 40) + 11, 1e-5
    x = (torch.randn(shape, generator=gen) + 5.0).to(xt)  # far from centred: the variance is no difference of large sums
    delta = None if dt is None else torch.randn(shape, generator=gen).to(dt)
    w, b = torch.randn(D, generator=gen), torch.randn(D, generator=gen)
    dy, dres = torch.randn(shape, generator=gen).to(yt), torch.randn(shape, generator=gen)
    leaves = [None if t is None else t.to(DEV).requires_grad_(True) for t in (x, delta, w, b)]
    xg, dg, wg, bg = leaves
    leaves = [t for t in leaves if t is not None]
    if delta is None:
        xn, y = None, layer_norm(xg, wg, bg, yt, eps)
        grads = torch.autograd.grad(y, leaves, dy.to(DEV))
    else:
        xn, y = add_layer_norm(xg, dg, wg, bg, yt, eps, p, seed, 2)
        grads = torch.autograd.grad((xn, y), leaves, (dres.to(DEV), dy.to(DEV)))
    assert y.dtype == yt and all(a.dtype == t.dtype for a, t in zip(grads, leaves))

    ref = [None if t is None else t.double().requires_grad_(True) for t in (x, delta, w, b)]
    rxn, ry = _reference(*ref, None if delta is None else _factor(shape, p, seed, 2), eps)
    ref = [t for t in ref if t is not None]
    rgrads = torch.autograd.grad((rxn, ry) if delta is not None else ry, ref,
                                 (dres.double(), dy.double()) if delta is not None else dy.double())
    if delta is not None:
        assert xn.dtype == f32 and _rel(xn, rxn) <= F32
    # a row's (x - mean) / sigma has the size of 1; x's rounding to fp32 at 5 + xi is 2^-22
    if D > 1:
        assert _rel(y, ry) <= _tol(yt)
    for name, g, r, t in zip(("x", "delta", "w", "b") if delta is not None else ("x", "w", "b"), grads, rgrads, leaves):
        if D == 1 and name in ("x", "w") and delta is None:
            assert float(g.abs().max()) <= 1e-2  # (exactly zero in float64: rows of one value are constant)
            continue
        lim = _tol(t.dtype)
        assert _rel(g, r) <= lim, f"d{name}: {_rel(g, r):.2e} > {lim:.1e}"


def test_layer_norm_strided_and_without_bias():
    from gruboros_amd.norm import layer_norm

    gen = torch.Generator().manual_seed(0)
    big = torch.randn(6, 40, 2 * 96, generator=gen)
    x = big.to(DEV)[1::2, ::3, 96:].requires_grad_(True)
    w = torch.randn(96, generator=gen).to(DEV).to(bf16).requires_grad_(True)  # a weight of another dtype
    y = layer_norm(x, w)
    dx, dw = torch.autograd.grad(y, (x, w), torch.ones_like(y).expand_as(y))
    rx, rw = big[1::2, ::3, 96:].double().requires_grad_(True), w.detach().double().cpu().requires_grad_(True)
    _, ry = _reference(rx, None, rw, None, None, 1e-5)
    rdx, rdw = torch.autograd.grad(ry, (rx, rw), torch.ones_like(ry))
    assert _rel(y, ry) <= F32 and dw.dtype == bf16 and _rel(dw, rdw) <= BF16
    assert float((dx.double().cpu() - rdx).abs().max()) <= F32  # (a sum to zero of terms of the size of 1)


def test_dropped_values_are_the_same_everywhere():
    """add_layer_norm drops what dropout drops, and the words are the oracle's, beyond 2^32 of a counter too."""
    from gruboros_amd.dropout import dropout
    from gruboros_amd.norm import add_layer_norm

    assert philox.block((0, 0, 0, 0), (0, 0)) == [0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8]
    assert philox.block((0xFFFFFFFF,) * 4, (0xFFFFFFFF,) * 2) == [0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD]
    for D in (96, 97):
        x, delta = torch.zeros(1, 50, D, device=DEV), torch.ones(1, 50, D, device=DEV)
        seed, offset = (1 << 63) + 5, (1 << 40) + 1
        want = _factor((1, 50, D), 0.4, seed, offset)
        xn, _ = add_layer_norm(x, delta, torch.ones(D, device=DEV), dropout_p=0.4, seed=seed, offset=offset)
        assert torch.equal(xn.cpu(), want.float())
        assert torch.equal(dropout(delta, 0.4, seed, offset).cpu(), want.float())


@pytest.mark.parametrize("n", [1, 7, 8, 1001, 70000])
@pytest.mark.parametrize("types", [(f32, None), (bf16, None), (bf16, f32), (f32, f32), (bf16, bf16)],
                         ids=lambda t: "-".join("none" if x is None else str(x)[6:] for x in t))
def test_dropout(n, types):
    from gruboros_amd.dropout import dropout

    xt, rt = types
    gen = torch.Generator().manual_seed(n)
    x = torch.randn(n, generator=gen).to(xt)
    r = None if rt is None else torch.randn(n, generator=gen).to(rt)
    yt = xt if rt is None else rt
    dy = torch.randn(n, generator=gen).to(yt)
    p, seed = 0.1, 77
    leaves = [t.to(DEV).requires_grad_(True) for t in (x, r) if t is not None]
    y = dropout(leaves[0], p, seed, 5, leaves[1] if r is not None else None)
    grads = torch.autograd.grad(y, leaves, dy.to(DEV))
    f = _factor((n,), p, seed, 5)
    want = x.double() * f + (0 if r is None else r.double())
    assert y.dtype == yt and _rel(y, want) <= (2.0 ** -23 if yt == f32 else 2.0 ** -8 + 2.0 ** -23)
    assert _rel(grads[0], dy.double() * f) <= (2.0 ** -23 if xt == f32 else 2.0 ** -8 + 2.0 ** -23)
    if r is not None:
        assert torch.equal(grads[1].cpu(), dy)
    # a dropped value is 0 whatever it was
    x2 = torch.where(f == 0, torch.tensor(float("nan")), x.float()).to(xt)
    assert torch.equal(dropout(x2.to(DEV), p, seed, 5), dropout(x.to(DEV), p, seed, 5))


def test_dropout_share():
    """A share of p is dropped: of 10^6 values within 5 sigma."""
    from gruboros_amd.dropout import dropout

    for p in (0.0, 0.1, 0.5, 0.999):
        kept = float((dropout(torch.ones(10 ** 6, device=DEV), p, 3) != 0).double().mean())
        assert abs(kept - (1 - p)) <= 5 * (p * (1 - p) / 10 ** 6) ** 0.5


def test_seed_tensor_in_a_graph():
    """A captured step reads the seed when it is replayed: each replay drops what an eager call with
    the same seed drops, in the forward and the backward."""
    from gruboros_amd.norm import add_layer_norm

    gen = torch.Generator().manual_seed(1)
    x, d = (torch.randn(4, 70, 96, generator=gen).to(DEV).requires_grad_(True) for _ in range(2))
    w = torch.randn(96, generator=gen).to(DEV).requires_grad_(True)
    dy = torch.randn(4, 70, 96, generator=gen).to(DEV)
    seed = torch.zeros(1, dtype=torch.int64, device=DEV)

    def step(s):
        xn, y = add_layer_norm(x, d, w, dropout_p=0.3, seed=s, offset=1)
        return [xn, y, *torch.autograd.grad((xn, y), (x, d, w), (dy, dy))]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(seed)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(seed)
    for k in (5, 6, 1 << 40):
        want = step(k)
        seed.fill_(k)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want))


def test_refusals():
    from gruboros_amd._lib import MingruHipError
    from gruboros_amd.dropout import dropout
    from gruboros_amd.norm import add_layer_norm, layer_norm

    x, w = torch.zeros(2, 8, device=DEV), torch.ones(8, device=DEV)
    for bad in (dict(p=1.0), dict(p=-0.1), dict(seed=None), dict(seed=-1), dict(seed=1 << 64), dict(offset=-1),
                dict(seed=torch.zeros(2, dtype=torch.int64, device=DEV)), dict(seed=torch.zeros(1, dtype=torch.int64)),
                dict(residual=torch.zeros(2, 9, device=DEV)), dict(residual=x.bfloat16())):
        with pytest.raises(ValueError):
            dropout(x, **{"p": 0.1, "seed": 1, **bad})
    with pytest.raises(MingruHipError):
        dropout(x.half(), 0.1, 1)
    with pytest.raises(ValueError):
        add_layer_norm(x, x, w, dropout_p=0.1)  # no seed
    with pytest.raises(ValueError):
        add_layer_norm(x.bfloat16(), x, w)
    with pytest.raises(ValueError):
        layer_norm(x, torch.ones(9, device=DEV))
    with pytest.raises(ValueError):
        layer_norm(torch.zeros(1, 16385, device=DEV), torch.ones(16385, device=DEV))
    assert layer_norm(torch.zeros(0, 8, device=DEV), w).shape == (0, 8) and dropout(x[:0], 0.1, 1).shape == (0, 8)
    y = dropout(x.requires_grad_(True), 0.1, 1)
    (g,) = torch.autograd.grad(y.sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()
