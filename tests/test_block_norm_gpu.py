"""The norms around a block with its gate and residual scale (add_gated_rms_norm) against float64.

Tolerances before any run. float32: a row's sum of squares has terms of one sign and trees of at most
16 values of a lane, 6 lane steps and 16 waves, 38 * 2^-24 = 2.3e-6 of it, half of that in its root;
the gate's exp and reciprocal 2^-22 for |gate| <= 8; the backward passes two such sums after them:
1e-5. Weight gradients: sums over rows, workgroups and partial rows of the same depth: 1e-5 of the
terms' size, which is the sums' own for random terms up to a factor of 2: 2e-5. bfloat16: half a
step, 2^-8 of each value, on top.
"""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
f32, bf16 = torch.float32, torch.bfloat16
F32, SUM = 1e-5, 2e-5
EPS = 1e-6


def _tol(dtype):
    return F32 + (2.0 ** -8 if dtype == bf16 else 0.0)


def _rel(a, b):
    a, b = a.detach().double().cpu(), b.detach().double().cpu()
    return float((a - b).norm() / b.norm().clamp_min(1e-30))


def _reference(x, branch, w_branch, w, gate, scale, activation, eps=EPS):
    def norm(t):
        return t / (t.square().mean(-1, keepdim=True) + eps).sqrt()

    b = norm(branch) * w_branch
    if gate is not None:
        b = b * torch.sigmoid(gate) * (gate if activation == "silu" else 1.0)
    xn = x + (b if scale is None else scale * b)
    return xn, norm(xn) * w


def _operands(shape, ft, gated, scaled, seed=0):
    gen = torch.Generator().manual_seed(seed + sum(shape))
    n = lambda *s: torch.randn(*s, generator=gen)  # noqa: E731
    D = shape[-1]
    return {"x": 2.0 * n(*shape), "branch": (3.0 * n(*shape)).to(ft), "w_branch": 1.0 + 0.2 * n(D), "w": 1.0 + 0.2 * n(D),
            "gate": (2.0 * n(*shape)).to(ft) if gated else None, "scale": 0.5 + 0.2 * n(D) if scaled else None}, n(*shape), n(*shape)


def _compare(ops, dres, dy, activation, yt, change=lambda k, t: t):
    from gruboros_amd.norm import add_gated_rms_norm

    dev = {k: None if t is None else change(k, t.to(DEV)).requires_grad_(True) for k, t in ops.items()}
    ref = {k: None if t is None else t.double().requires_grad_(True) for k, t in ops.items()}
    xn, y = add_gated_rms_norm(**dev, activation=activation, out_dtype=yt, eps=EPS)
    rxn, ry = _reference(**ref, activation=activation)
    assert xn.dtype == f32 and y.dtype == yt
    assert _rel(xn, rxn) <= F32 and _rel(y, ry) <= _tol(yt)
    names = [k for k, t in ops.items() if t is not None]
    up = dy.to(yt)
    grads = torch.autograd.grad((xn, y), [dev[k] for k in names], (dres.to(DEV), up.to(DEV)))
    want = torch.autograd.grad((rxn, ry), [ref[k] for k in names], (dres.double(), up.double()))
    D = ops["x"].shape[-1]
    for k, g, r in zip(names, grads, want):
        assert g.dtype == dev[k].dtype and g.shape == dev[k].shape
        if D == 1 and k == "branch":  # (f / |f| has a slope of eps only: what is left of a difference of ones)
            assert float((g.double().cpu() - r).abs().max()) <= 1e-5 * float(dres.abs().max() + dy.abs().max()) / float(
                ops["branch"].double().abs().min())
            continue
        lim = _tol(dev[k].dtype) if k in ("x", "branch", "gate") else SUM
        assert _rel(g, r) <= lim, f"d{k}: {_rel(g, r):.2e} > {lim:.1e}"


SHAPES = [(1, 1, 1), (2, 3, 7), (3, 5, 64), (1, 130, 250), (1, 9, 257), (2, 33, 1024), (1, 9, 1001), (1, 3, 1025), (2, 5, 2048), (1, 7, 2500),
          (1, 5, 4095), (1, 5, 4097), (1, 3, 9000), (1, 2, 16384), (5000, 1, 24)]


@pytest.mark.parametrize("types", [(f32, f32), (bf16, bf16), (bf16, f32), (f32, bf16)], ids=lambda t: "-".join(str(x)[6:] for x in t))
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "x".join(map(str, s)))
@pytest.mark.parametrize("form", [("silu", True), ("sigmoid", False), (None, True), (None, False)], ids=lambda f: f"{f[0]}-{f[1]}")
def test_parity(shape, types, form):
    ft, yt = types
    ops, dres, dy = _operands(shape, ft, form[0] is not None, form[1])
    _compare(ops, dres, dy, form[0] or "silu", yt)


@pytest.mark.parametrize("shape", [(1, 4500, 260), (1, 1500, 1100), (2, 300, 4100), (1, 530, 8195), (1, 530, 12289)], ids=lambda s: "x".join(map(str, s)))
def test_more_rows_than_workgroups(shape):
    """Sums over several rows of one workgroup, of every number of threads to a row, and those kept in LDS."""
    for types in ((bf16, bf16), (f32, f32)):
        _compare(*_operands(shape, types[0], True, True), "silu", types[1])


def test_views():
    """Columns of wider tensors at odd offsets, transposed batch, weights of other types."""
    ops, dres, dy = _operands((6, 10, 97), bf16, True, True)

    def change(k, t):
        if t.dim() == 1:
            return t
        wide = torch.zeros(10, 6, 2 * 97 + 1, dtype=t.dtype, device=DEV)
        wide[..., 98:] = t.transpose(0, 1)
        return wide[..., 98:].transpose(0, 1).detach()

    _compare(ops, dres, dy, "silu", bf16, change)


def test_weights_of_other_types_and_a_broadcast_gate():
    from gruboros_amd.norm import add_gated_rms_norm

    ops, dres, dy = _operands((4, 6, 40), f32, True, True)
    ops["gate"] = ops["gate"][:, :1].contiguous()
    for k in ("w_branch", "w", "scale"):
        ops[k] = ops[k].to(bf16)
    dev = {k: t.to(DEV).requires_grad_(True) for k, t in ops.items()}
    ref = {k: t.double().requires_grad_(True) for k, t in ops.items()}
    out = add_gated_rms_norm(**dev, activation="sigmoid", eps=EPS)
    rout = _reference(**ref, activation="sigmoid")
    grads = torch.autograd.grad(out, list(dev.values()), (dres.to(DEV), dy.to(DEV)))
    want = torch.autograd.grad(rout, list(ref.values()), (dres.double(), dy.double()))
    for k, g, r in zip(dev, grads, want):
        assert g.shape == dev[k].shape and g.dtype == dev[k].dtype and _rel(g, r) <= _tol(g.dtype) + SUM, k


def test_against_differences():
    from gruboros_amd.norm import add_gated_rms_norm

    ops, dres, dy = _operands((2, 9, 70), f32, True, True)
    dev = {k: t.to(DEV).requires_grad_(True) for k, t in ops.items()}
    out = add_gated_rms_norm(**dev, eps=EPS)
    grads = torch.autograd.grad(out, list(dev.values()), (dres.to(DEV), dy.to(DEV)))
    base = {k: t.double() for k, t in ops.items()}

    def value(o):
        xn, y = _reference(**o, activation="silu")
        return float((xn * dres.double()).sum() + (y * dy.double()).sum())

    gen, h = torch.Generator().manual_seed(1), 1e-5
    for (k, v), g in zip(base.items(), grads):
        d = torch.randn(v.shape, generator=gen, dtype=torch.float64)
        diff = (value({**base, k: v + h * d}) - value({**base, k: v - h * d})) / (2 * h)
        # (the gradient's 2e-5 of itself along a random direction; the difference: h^2 of third derivatives, 2^-53 / h)
        assert abs(float((g.double().cpu() * d).sum()) - diff) <= 2e-5 * float(g.double().norm()) * 4 + 1e-6, k


def test_rows_at_their_ends():
    """Rows of zeros, of large and small values; gates at the ends of their range; NaN in one row only spoils it."""
    from gruboros_amd.norm import add_gated_rms_norm

    D = 1500
    gen = torch.Generator().manual_seed(2)
    x, f, g = (torch.randn(8, D, generator=gen) for _ in range(3))
    f[0] = 0.0
    f[1] *= 1e15
    f[2] *= 1e-15
    x[3] = 0.0
    f[3] = 0.0
    g[4], g[5] = -200.0, 200.0
    w = torch.ones(D)
    for act in ("silu", "sigmoid"):
        leaves = [t.to(DEV).requires_grad_(True) for t in (x, f, w, w, g)]
        xn, y = add_gated_rms_norm(*leaves, activation=act, eps=EPS)
        rxn, ry = _reference(x.double(), f.double(), 1.0, 1.0, g.double(), None, act)
        assert float((xn.detach().cpu().double() - rxn).abs().max()) <= F32 * float(rxn.abs().max())
        assert float((y.detach().cpu().double() - ry).abs().max()) <= F32 * float(ry.abs().max())
        clean = torch.autograd.grad((xn, y), leaves, (torch.ones_like(xn), torch.ones_like(y)))
        assert all(bool(torch.isfinite(t).all()) for t in clean)
        bad = f.clone()
        bad[6, 3] = float("nan")
        leaves[1] = bad.to(DEV).requires_grad_(True)
        xb, yb = add_gated_rms_norm(*leaves, activation=act, eps=EPS)
        keep = [0, 1, 2, 3, 4, 5, 7]
        assert torch.equal(xb[keep], xn[keep]) and torch.equal(yb[keep], y[keep]) and bool(torch.isnan(yb[6]).all())
        got = torch.autograd.grad((xb, yb), leaves, (torch.ones_like(xn), torch.ones_like(y)))
        for i in (0, 1, 4):
            assert torch.equal(got[i][keep], clean[i][keep])
    shut = torch.full_like(g, -float("inf")).to(DEV)
    xn, _ = add_gated_rms_norm(x.to(DEV), f.to(DEV), w.to(DEV), w.to(DEV), shut)
    assert torch.equal(xn.cpu(), x)


def test_only_some_gradients():
    from gruboros_amd.norm import add_gated_rms_norm

    ops, dres, dy = _operands((3, 11, 100), bf16, True, True)
    up = (dres.to(DEV), dy.to(bf16).to(DEV))
    full = {k: t.to(DEV).requires_grad_(True) for k, t in ops.items()}
    want = torch.autograd.grad(add_gated_rms_norm(**full, out_dtype=bf16), list(full.values()), up)
    for i, k in enumerate(ops):
        some = {n: t.to(DEV).requires_grad_(n == k) for n, t in ops.items()}
        assert torch.equal(torch.autograd.grad(add_gated_rms_norm(**some, out_dtype=bf16), some[k], up)[0], want[i])
    # the norm alone, the stream alone, and the two together
    xn, y = add_gated_rms_norm(**full)
    a = torch.autograd.grad(xn, list(full.values()), up[0], retain_graph=True, allow_unused=True)
    b = torch.autograd.grad(y, list(full.values()), dy.to(DEV), retain_graph=True)
    both = torch.autograd.grad((xn, y), list(full.values()), (up[0], dy.to(DEV)))
    zero = [torch.zeros_like(t) if s is None else s for t, s in zip(full.values(), a)]
    for k, p, q, r in zip(full, zero, b, both):
        assert _rel(p.double() + q.double(), r) <= 3 * _tol(r.dtype), k
    (gx,) = torch.autograd.grad(add_gated_rms_norm(**full)[1].sum(), full["x"], create_graph=True)
    with pytest.raises(RuntimeError):
        gx.sum().backward()


def test_no_values():
    from gruboros_amd.norm import add_gated_rms_norm

    leaves = [torch.zeros(*s, device=DEV).requires_grad_(True) for s in ((0, 16), (0, 16), (16,), (16,), (0, 16), (16,))]
    xn, y = add_gated_rms_norm(*leaves[:5], scale=leaves[5], out_dtype=bf16)
    assert y.dtype == bf16
    for out in (xn, y):
        grads = torch.autograd.grad(out.sum(), leaves, retain_graph=True)
        assert all(g.shape == t.shape and bool((g == 0).all()) for g, t in zip(grads, leaves))


def test_streams_and_graphs():
    from gruboros_amd.norm import add_gated_rms_norm

    made = []
    for seed in (0, 1):
        ops, dres, dy = _operands((3, 200, 384), bf16, True, True, seed)
        leaves = {k: t.to(DEV).requires_grad_(True) for k, t in ops.items()}
        up = (dres.to(DEV), dy.to(bf16).to(DEV))

        def call(leaves=leaves, up=up):
            out = add_gated_rms_norm(**leaves, out_dtype=bf16)
            return [*(t.detach() for t in out), *torch.autograd.grad(out, list(leaves.values()), up)]

        side = torch.cuda.Stream()
        with torch.cuda.stream(side):
            call()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = call()
        made.append((graph, out, leaves, call))
    gen = torch.Generator(device=DEV).manual_seed(3)
    for _ in range(4):
        for graph, out, leaves, call in made:
            with torch.no_grad():
                leaves["x"].copy_(torch.randn(leaves["x"].shape, generator=gen, device=DEV))
            graph.replay()
            torch.cuda.synchronize()
            got = [t.clone() for t in out]
            assert all(torch.equal(a, b) for a, b in zip(got, call()))
    want = [m[3]() for m in made]
    torch.cuda.synchronize()
    for _ in range(3):
        for m in made:
            with torch.cuda.stream(torch.cuda.Stream()):
                m[0].replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for w, m in zip(want, made) for a, b in zip(m[1], w))


def test_values_beyond_32_bit_offsets():
    from gruboros_amd.norm import add_gated_rms_norm

    D = 1023
    N = 2 ** 31 // D + 40
    gen = torch.Generator(device=DEV).manual_seed(0)
    x = torch.randn(N, D, generator=gen, device=DEV)
    f = torch.randn(N, D, generator=gen, device=DEV, dtype=bf16)
    w = torch.ones(D, device=DEV)
    leaves = [x.requires_grad_(True), f.requires_grad_(True)]
    xn, y = add_gated_rms_norm(*leaves, w, w, gate=f.detach(), out_dtype=bf16)
    g = torch.autograd.grad((xn, y), leaves, (xn.detach(), f.detach()))
    for part in (slice(0, 9), slice(N - 9, N)):
        few = [t.detach()[part].clone().requires_grad_(True) for t in (x, f)]
        a, b = add_gated_rms_norm(*few, w, w, gate=f.detach()[part], out_dtype=bf16)
        assert torch.equal(a, xn[part]) and torch.equal(b, y[part])
        h = torch.autograd.grad((a, b), few, (a.detach(), f.detach()[part]))
        assert all(torch.equal(p, q[part]) for p, q in zip(h, g))


@pytest.mark.parametrize("grad", [True, False], ids=["grad", "no grad"])
def test_dual_tensors_are_refused(grad):
    import torch.autograd.forward_ad as fwd

    from gruboros_amd.norm import add_gated_rms_norm

    ops = {k: t.to(DEV) for k, t in _operands((3, 16), f32, True, True)[0].items()}
    with torch.set_grad_enabled(grad), fwd.dual_level():
        for k, t in ops.items():
            with pytest.raises((RuntimeError, NotImplementedError)):
                add_gated_rms_norm(**{**ops, k: fwd.make_dual(t, torch.ones_like(t))})
        add_gated_rms_norm(**ops)


def test_refusals():
    from gruboros_amd._lib import MingruHipError
    from gruboros_amd.norm import add_gated_rms_norm

    ops = {k: t.to(DEV) for k, t in _operands((3, 5, 16), f32, True, True)[0].items()}
    for bad in (dict(x=ops["x"].bfloat16()), dict(branch=ops["branch"][:2]), dict(w=ops["w"][:15]), dict(w_branch=ops["w"].int()),
                dict(scale=ops["x"]), dict(gate=ops["gate"].bfloat16()), dict(gate=ops["gate"][:2]), dict(gate=ops["gate"][None, None]),
                dict(activation="gelu"), dict(eps=-1.0), dict(eps=float("nan")), dict(x=torch.zeros(2, 16385, device=DEV))):
        with pytest.raises(ValueError):
            add_gated_rms_norm(**{**ops, **bad})
    for bad in (dict(branch=ops["branch"].half(), gate=ops["gate"].half()), dict(out_dtype=torch.float16), dict(w=torch.ones(16))):
        with pytest.raises(MingruHipError):
            add_gated_rms_norm(**{**ops, **bad})
