"""The gated linear recurrence against its definition in float64.

Tolerances before any run. float32: a step's factor and addend are off by at most 4 half steps each
(2^-22: exp, two reciprocals, a root, the products); over the T <= 2100 steps that a state can hold
on to, errors of either sign add like a root, 46 * 2^-22 = 1.1e-5, and the backward passes through
both scans: 2e-5. bfloat16: half a step, 2^-8 of each value, on top. Sums over all steps (decay):
their terms' errors of 2e-5 and the sums' own, at most 300 terms in a row, 300 * 2^-24 = 1.8e-5: 4e-5
of the size of the terms' sum in one sign.
"""
import pytest
import torch

from oracle.recurrence_oracle import gated_recurrence as oracle

pytestmark = pytest.mark.gpu
DEV = "cuda"
f32, bf16 = torch.float32, torch.bfloat16
TOL = {f32: 2e-5, bf16: 2.0 ** -8 + 2e-5}
NAMES = ("x", "input_gate", "decay_gate", "decay", "initial_state")


def _rel(a, b):
    a, b = a.detach().double().cpu(), b.detach().double().cpu()
    return float((a - b).norm() / b.norm().clamp_min(1e-30))


def _operands(B, T, D, dtype, seed=0, carried=True, packed=False):
    gen = torch.Generator().manual_seed(seed + 1000 * T + D)
    n = lambda *s: torch.randn(*s, generator=gen)  # noqa: E731
    rate = -torch.log(0.9 + 0.099 * torch.rand(D, generator=gen)) / 8.0
    ops = {"x": n(B, T, D).to(dtype), "input_gate": n(B, T, D).to(dtype), "decay_gate": n(B, T, D).to(dtype),
           "decay": torch.log(torch.expm1(rate)), "initial_state": n(B, D) if carried else None}
    reset = (torch.rand(B, T, generator=gen) < 0.02) if packed else None
    return ops, reset, n(B, T, D).to(dtype), n(B, D)


def _reference(ops, reset, dh, dlast):
    r = {k: None if v is None else v.double().requires_grad_(True) for k, v in ops.items()}
    h, last = oracle(**r, reset=reset)
    leaves = [v for v in r.values() if v is not None]
    loss = (h * dh.double()).sum() + (0 if dlast is None else (last * dlast.double()).sum())
    grads = torch.autograd.grad(loss, leaves)
    return h, last, dict(zip([k for k, v in r.items() if v is not None], grads))


def _compare(ops, reset, dh, dlast, dtype, views=lambda t: t):
    from gruboros_amd.recurrence import gated_recurrence

    h_ref, last_ref, g_ref = _reference(ops, reset, dh, dlast)
    dev = {k: None if v is None else views(v.to(DEV)).requires_grad_(True) for k, v in ops.items()}
    mark = None if reset is None else reset.to(DEV)
    h, last = gated_recurrence(**dev, reset=mark, return_state=True)
    assert h.dtype == dtype and last.dtype == f32
    assert _rel(h, h_ref) <= TOL[dtype] and _rel(last, last_ref) <= TOL[f32]
    leaves = {k: v for k, v in dev.items() if v is not None}
    outs, up = [h], [dh.to(DEV)]
    if dlast is not None:
        outs.append(last), up.append(dlast.to(DEV))
    for (k, t), g in zip(leaves.items(), torch.autograd.grad(outs, list(leaves.values()), up)):
        assert g.dtype == t.dtype and g.shape == t.shape
        lim = 4e-5 if k == "decay" else TOL[t.dtype]
        if k == "decay":  # of the size of its terms' sum in one sign
            err = (g.double().cpu() - g_ref[k]).norm()
            size = g_ref[k].norm() * max(1.0, (dh.shape[0] * dh.shape[1]) ** 0.5 / 8)
            assert float(err) <= lim * float(size), f"d{k}"
        elif float(g_ref[k].norm()) == 0.0:
            assert float(g.abs().max()) == 0.0, f"d{k}"
        else:
            assert _rel(g, g_ref[k]) <= lim, f"d{k}: {_rel(g, g_ref[k]):.2e}"


@pytest.mark.parametrize("dtype", [f32, bf16], ids=["f32", "bf16"])
@pytest.mark.parametrize("size", [(1, 1, 1), (2, 3, 5), (3, 7, 64), (1, 8, 63), (2, 9, 65), (1, 64, 130), (2, 65, 96), (1, 127, 1),
                                  (2, 128, 66), (1, 129, 40), (3, 300, 70), (1, 2100, 24)], ids=lambda s: "x".join(map(str, s)))
@pytest.mark.parametrize("form", ["plain", "carried", "packed"])
def test_parity(size, dtype, form):
    ops, reset, dh, dlast = _operands(*size, dtype, carried=form != "plain", packed=form == "packed")
    _compare(ops, reset, dh, dlast if form != "plain" else None, dtype)


def test_every_token_a_sequence():
    ops, _, dh, dlast = _operands(2, 150, 20, f32)
    _compare(ops, torch.ones(2, 150, dtype=torch.bool), dh, dlast, f32)
    _compare(ops, torch.zeros(2, 150, dtype=torch.uint8), dh, dlast, f32)


def test_views_of_a_projection():
    """x and the gates as columns of one packed projection, at odd offsets, batch and steps swapped."""
    from gruboros_amd.recurrence import gated_recurrence, gated_recurrence_step

    ops, reset, dh, _ = _operands(2, 140, 37, bf16, packed=True)
    packed = torch.zeros(140, 2, 3 * 37 + 1, dtype=bf16)
    for i, k in enumerate(NAMES[:3]):
        packed[..., 1 + 37 * i:1 + 37 * (i + 1)] = ops[k].transpose(0, 1)
    packed = packed.to(DEV).requires_grad_(True)
    cols = [packed[..., 1 + 37 * i:1 + 37 * (i + 1)].transpose(0, 1) for i in range(3)]
    h = gated_recurrence(*cols, ops["decay"].to(DEV), ops["initial_state"].to(DEV), reset.to(DEV))
    (g,) = torch.autograd.grad(h, packed, dh.to(DEV))
    h_ref, _, g_ref = _reference(ops, reset, dh, None)
    assert _rel(h, h_ref) <= TOL[bf16] and float(g[..., 0].abs().max()) == 0.0
    for i, k in enumerate(NAMES[:3]):
        assert _rel(g[..., 1 + 37 * i:1 + 37 * (i + 1)].transpose(0, 1), g_ref[k]) <= TOL[bf16]
    # a gradient that is broadcast
    x = ops["x"].to(DEV).requires_grad_(True)
    args = [x, *(ops[k].to(DEV) for k in NAMES[1:4])]
    one = torch.autograd.grad(gated_recurrence(*args).sum(), x)[0]
    assert torch.equal(one, torch.autograd.grad(gated_recurrence(*args), x, torch.ones_like(x))[0])
    # a step on rows of the packed projection is the sequence's step
    state = ops["initial_state"].to(DEV).clone()
    with torch.no_grad():
        o = gated_recurrence_step(*(c[:, 0] for c in cols), ops["decay"].to(DEV), state)
        whole, last = gated_recurrence(*(c[:, :1] for c in cols), ops["decay"].to(DEV), ops["initial_state"].to(DEV), return_state=True)
    assert torch.equal(o, whole[:, 0]) and torch.equal(state, last)


@pytest.mark.parametrize("dtype", [f32, bf16], ids=["f32", "bf16"])
@pytest.mark.parametrize("B,D", [(1, 1), (3, 65), (130, 257), (2, 1024)])
def test_step(B, D, dtype):
    """Tokens one by one are the sequence; the state's version is bumped."""
    from gruboros_amd.recurrence import gated_recurrence, gated_recurrence_step

    ops, _, _, _ = _operands(B, 5, D, dtype)
    ops = {k: v.to(DEV) for k, v in ops.items()}
    h, last = gated_recurrence(**ops, return_state=True)
    state = ops["initial_state"].clone()
    v = state._version
    for t in range(5):
        o = gated_recurrence_step(ops["x"][:, t], ops["input_gate"][:, t], ops["decay_gate"][:, t], ops["decay"], state)
        assert o.dtype == dtype and _rel(o, h[:, t]) <= TOL[dtype]
    assert state._version == v + 5 and _rel(state, last) <= TOL[f32]
    a, r = (t.expand(B, D).contiguous() for t in (ops["x"][:1, 0], ops["decay"]))
    wide = torch.stack([a, a], -1)[..., 0]  # (a stride of two between channels)
    s1, s2 = state.clone(), state.clone()
    assert torch.equal(gated_recurrence_step(wide, a, a, r[0].bfloat16(), s1), gated_recurrence_step(a, a, a, r[0].bfloat16().float(), s2))
    assert torch.equal(s1, s2)


def test_gates_at_their_ends():
    """Shut and open gates: exact where a float32 sigmoid is 0, finite gradients, the oracle's state."""
    from gruboros_amd.recurrence import gated_recurrence

    inf = float("inf")
    vals = torch.tensor([-inf, -200.0, -90.0, -40.0, -20.0, 0.0, 20.0, 90.0, inf])
    D = len(vals)
    x = torch.randn(1, 140, D, generator=torch.Generator().manual_seed(3))
    for decay in (-100.0, -20.0, 0.0, 3.0, 30.0):
        dec = torch.full((D,), decay)
        gr = vals.expand(1, 140, D).contiguous()
        gi = torch.zeros(1, 140, D)
        h0 = torch.ones(1, D)
        leaves = [t.to(DEV).requires_grad_(True) for t in (x, gi, gr, dec, h0)]
        h = gated_recurrence(*leaves)
        ref, _ = oracle(x.double(), gi.double(), gr.double(), dec.double(), h0.double())
        err = (h.detach().cpu().double() - ref).abs().max()
        assert float(err) <= 2e-5 * float(ref.abs().max()), decay
        assert torch.equal(h[..., 0], torch.ones_like(h[..., 0]))  # a shut gate holds the state
        for g in torch.autograd.grad(h.sum(), leaves):
            assert bool(torch.isfinite(g).all())
    gi = vals.expand(1, 140, D).contiguous().to(DEV)
    h = gated_recurrence(x.to(DEV), gi, torch.zeros_like(gi), torch.zeros(D, device=DEV))
    assert bool((h[..., 0] == 0).all()) and bool(torch.isfinite(h).all())


@pytest.mark.parametrize("dtype", [f32, bf16], ids=["f32", "bf16"])
def test_what_is_not_finite_stays_in_its_sequence(dtype):
    from gruboros_amd.recurrence import gated_recurrence

    B, T, D = 2, 400, 70
    ops, _, dh, _ = _operands(B, T, D, dtype)
    reset = torch.zeros(B, T, dtype=torch.bool)
    reset[:, [0, 50, 137, 300, 301]] = True
    clean = {k: v.to(DEV) for k, v in ops.items()}
    h = gated_recurrence(**clean, reset=reset.to(DEV))
    bad = {k: v.clone() for k, v in ops.items()}
    bad["initial_state"][:] = float("nan")
    for name, at, v in (("x", 60, "nan"), ("x", 310, "inf"), ("decay_gate", 130, "nan"), ("input_gate", 70, "nan")):
        bad[name][:, at] = float(v)
    bad = {k: v.to(DEV).requires_grad_(True) for k, v in bad.items()}
    hb = gated_recurrence(**bad, reset=reset.to(DEV))
    for lo, hi in ((0, 60), (137, 310)):
        assert torch.equal(hb[:, lo:hi], h[:, lo:hi])
    assert bool(torch.isnan(hb[:, 60:137]).all())
    good = {k: v.clone().requires_grad_(True) for k, v in clean.items()}
    hg = gated_recurrence(**good, reset=reset.to(DEV))
    up = dh.to(DEV)
    spoilt = up.clone()
    spoilt[:, 250] = float("nan")  # a gradient spoils its own sequence only
    g1 = torch.autograd.grad(hg, [good[k] for k in NAMES], up)
    g2 = torch.autograd.grad(hb, [bad[k] for k in NAMES], spoilt)
    for a, b in zip(g1[:3], g2[:3]):
        assert torch.equal(a[:, :50], b[:, :50]) and torch.equal(a[:, 251:300], b[:, 251:300]) and torch.equal(a[:, 300], b[:, 300])
    assert torch.equal(g2[4], torch.zeros_like(g2[4])) and bool(torch.isnan(g2[0][:, 200]).all())


def test_against_differences():
    """The kernels' gradients against central differences of the definition in float64, along random directions."""
    from gruboros_amd.recurrence import gated_recurrence

    ops, reset, dh, dlast = _operands(2, 90, 33, f32, packed=True)
    dev = {k: v.to(DEV).requires_grad_(True) for k, v in ops.items()}
    h, last = gated_recurrence(**dev, reset=reset.to(DEV), return_state=True)
    grads = torch.autograd.grad([h, last], list(dev.values()), [dh.to(DEV), dlast.to(DEV)])

    def value(**o):
        h, last = oracle(**o, reset=reset)
        return float((h * dh.double()).sum() + (last * dlast.double()).sum())

    gen, eps = torch.Generator().manual_seed(5), 1e-5
    base = {k: v.double() for k, v in ops.items()}
    for (k, v), g in zip(base.items(), grads):
        d = torch.randn(v.shape, generator=gen, dtype=torch.float64)
        diff = (value(**{**base, k: v + eps * d}) - value(**{**base, k: v - eps * d})) / (2 * eps)
        size = float(g.double().cpu().norm() * d.norm())
        # (the difference itself: eps^2 of third derivatives, and rounding 2^-53 / eps of the value)
        assert abs(float((g.double().cpu() * d).sum()) - diff) <= 1e-4 * size / v.numel() ** 0.5 + 1e-6, k


def test_only_some_gradients():
    from gruboros_amd.recurrence import gated_recurrence

    ops, _, dh, dlast = _operands(2, 70, 17, f32)
    full = {k: v.to(DEV).requires_grad_(True) for k, v in ops.items()}
    h, last = gated_recurrence(**full, return_state=True)
    want = torch.autograd.grad([h, last], list(full.values()), [dh.to(DEV), dlast.to(DEV)])
    for i, k in enumerate(NAMES):
        some = {n: v.to(DEV).requires_grad_(n == k) for n, v in ops.items()}
        h, last = gated_recurrence(**some, return_state=True)
        assert torch.equal(torch.autograd.grad([h, last], some[k], [dh.to(DEV), dlast.to(DEV)])[0], want[i])
    # the state alone; neither
    full = {k: v.to(DEV).requires_grad_(True) for k, v in ops.items()}
    h, last = gated_recurrence(**full, return_state=True)
    g = torch.autograd.grad(last, list(full.values()), dlast.to(DEV), retain_graph=True)
    _, _, ref = _reference(ops, None, torch.zeros_like(dh), dlast)
    assert all(_rel(a, ref[k]) <= 4e-5 for a, k in zip(g, NAMES))
    # run again, the same bits; a second derivative is refused
    again = torch.autograd.grad(last, list(full.values()), dlast.to(DEV))
    assert all(torch.equal(a, b) for a, b in zip(g, again))
    h = gated_recurrence(**full)
    (gx,) = torch.autograd.grad(h.sum(), full["x"], create_graph=True)
    with pytest.raises(RuntimeError):
        gx.sum().backward()


def test_decay_of_another_type():
    from gruboros_amd.recurrence import gated_recurrence

    ops, _, dh, _ = _operands(1, 40, 16, bf16)
    dev = {k: v.to(DEV) for k, v in ops.items()}
    d = dev["decay"].to(bf16).requires_grad_(True)
    h = gated_recurrence(**{**dev, "decay": d})
    assert torch.equal(h, gated_recurrence(**{**dev, "decay": d.detach().float()}))
    assert torch.autograd.grad(h, d, dh.to(DEV))[0].dtype == bf16


@pytest.mark.parametrize("size", [(0, 4, 8), (2, 0, 8), (2, 4, 0)], ids=str)
def test_no_values(size):
    from gruboros_amd.recurrence import gated_recurrence, gated_recurrence_step

    B, T, D = size
    leaves = [torch.zeros(size, device=DEV).requires_grad_(True) for _ in range(3)]
    leaves += [torch.zeros(D, device=DEV).requires_grad_(True), torch.ones(B, D, device=DEV).requires_grad_(True)]
    h, last = gated_recurrence(*leaves, return_state=True)
    assert h.shape == size and torch.equal(last, leaves[4])
    g = torch.autograd.grad(h.sum(), leaves, retain_graph=True)
    assert all(bool((t == 0).all()) for t in g)
    assert torch.equal(torch.autograd.grad(last.sum(), leaves[4])[0], torch.ones(B, D, device=DEV))
    with torch.no_grad():
        if T:
            assert gated_recurrence_step(*(t[:, 0] for t in leaves[:3]), leaves[3], leaves[4].clone()).shape == (B, D)


def test_streams_and_overlapping_calls():
    """Calls on two streams at once, workspaces and all, give the bits of calls alone."""
    from gruboros_amd.recurrence import gated_recurrence

    sets = [{k: v.to(DEV) for k, v in _operands(4, 1000, 256, bf16, seed=s)[0].items()} for s in range(2)]
    want = [gated_recurrence(**o) for o in sets]
    streams = [torch.cuda.Stream() for _ in sets]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(6):
        for i, (s, o) in enumerate(zip(streams, sets)):
            with torch.cuda.stream(s):
                got[i].append(gated_recurrence(**o))
    torch.cuda.synchronize()
    assert all(torch.equal(g, want[i]) for i in range(2) for g in got[i])


def test_captured_passes():
    """Two captured passes, replayed between eager calls and at once on two streams; training and steps."""
    from gruboros_amd.recurrence import gated_recurrence, gated_recurrence_step

    made = []
    for seed in (0, 1):
        ops, reset, dh, _ = _operands(2, 700, 130, bf16, seed=seed, packed=True)
        leaves = {k: v.to(DEV).requires_grad_(True) for k, v in ops.items()}
        reset, dh = reset.to(DEV), dh.to(DEV)

        def call(leaves=leaves, reset=reset, dh=dh):
            h = gated_recurrence(**leaves, reset=reset)
            return [h.detach(), *torch.autograd.grad(h, list(leaves.values()), dh)]

        side = torch.cuda.Stream()
        with torch.cuda.stream(side):
            call()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = call()
        made.append((graph, out, leaves, call))
    gen = torch.Generator(device=DEV).manual_seed(9)
    for rep in range(4):
        for graph, out, leaves, call in made:
            with torch.no_grad():
                leaves["x"].copy_(torch.randn(leaves["x"].shape, generator=gen, device=DEV))
            graph.replay()
            torch.cuda.synchronize()
            got = [t.clone() for t in out]
            assert all(torch.equal(a, b) for a, b in zip(got, call())), rep
    want = [call() for _, _, _, call in made]
    streams = [torch.cuda.Stream() for _ in made]
    torch.cuda.synchronize()
    for _ in range(3):
        for s, (graph, *_) in zip(streams, made):
            with torch.cuda.stream(s):
                graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for w, m in zip(want, made) for a, b in zip(m[1], w))
    ops = {k: v.to(DEV) for k, v in _operands(3, 1, 96, bf16)[0].items()}
    state, rows = ops["initial_state"].clone(), [ops[k][:, 0].contiguous() for k in NAMES[:3]]
    twin = state.clone()
    with torch.no_grad():
        gated_recurrence_step(*rows, ops["decay"], state.clone())
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            o = gated_recurrence_step(*rows, ops["decay"], state)
        for _ in range(4):
            graph.replay()
            assert torch.equal(o, gated_recurrence_step(*rows, ops["decay"], twin)) and torch.equal(state, twin)


def test_values_beyond_32_bit_offsets():
    """More than 2^31 values each way: every batch row of broadcast operands is the row alone."""
    from gruboros_amd.recurrence import gated_recurrence

    B, T, D = 33, 32771, 2000
    gen = torch.Generator(device=DEV).manual_seed(1)
    one = [torch.randn(1, T, D, generator=gen, device=DEV, dtype=bf16) for _ in range(4)]
    decay = torch.full((D,), -6.0, device=DEV)
    leaves = [t.clone().requires_grad_(True) for t in one[:3]]
    h1 = gated_recurrence(*leaves, decay)
    g1 = torch.autograd.grad(h1, leaves, one[3])
    wide = [t.expand(B, T, D).detach().requires_grad_(True) for t in one[:3]]
    h = gated_recurrence(*wide, decay)
    assert h.numel() > 2 ** 31
    g = torch.autograd.grad(h, wide, one[3].expand(B, T, D))
    for b in (0, 16, B - 2, B - 1):
        assert torch.equal(h[b], h1[0]) and all(torch.equal(a[b], r[0]) for a, r in zip(g, g1))


@pytest.mark.parametrize("grad", [True, False], ids=["grad", "no grad"])
def test_dual_tensors_are_refused(grad):
    import torch.autograd.forward_ad as fwd

    from gruboros_amd.recurrence import gated_recurrence, gated_recurrence_step

    ops = {k: v.to(DEV) for k, v in _operands(1, 4, 8, f32)[0].items()}
    tok = {k: v[:, 0].contiguous() if k in NAMES[:3] else v for k, v in ops.items()}
    tok["state"] = tok.pop("initial_state")
    with torch.set_grad_enabled(grad), fwd.dual_level():
        for call, operands in ((gated_recurrence, ops), (gated_recurrence_step, tok)):
            for n, t in operands.items():
                before = tok["state"].clone()
                with pytest.raises((RuntimeError, NotImplementedError)):
                    call(**{**operands, n: fwd.make_dual(t, torch.ones_like(t))})
                assert torch.equal(before, tok["state"])
            call(**operands)


def test_refusals():
    from gruboros_amd._lib import MingruHipError
    from gruboros_amd.recurrence import gated_recurrence, gated_recurrence_step

    ops = {k: v.to(DEV) for k, v in _operands(2, 6, 8, f32)[0].items()}
    x = ops["x"]
    bad = [dict(x=x[0]), dict(input_gate=x[:, :5]), dict(decay_gate=x.bfloat16()), dict(decay=ops["decay"][:7]), dict(decay=ops["decay"].int()),
           dict(initial_state=x[:, 0, :7]), dict(initial_state=x[:, 0].bfloat16()), dict(reset=torch.zeros(2, 5, device=DEV, dtype=torch.bool)),
           dict(reset=torch.zeros(2, 6, device=DEV)), dict(c=-1.0), dict(c=float("nan")), dict(c=float("inf"))]
    for b in bad:
        with pytest.raises(ValueError):
            gated_recurrence(**{**ops, **b})
    for b in (dict(x=x.half(), input_gate=x.half(), decay_gate=x.half()), dict(decay=ops["decay"].cpu()), dict(initial_state=torch.zeros(2, 8)),
              dict(reset=torch.zeros(2, 6, dtype=torch.bool))):
        with pytest.raises(MingruHipError):
            gated_recurrence(**{**ops, **b})
    row = dict(x=x[:, 0], input_gate=x[:, 0], decay_gate=x[:, 0], decay=ops["decay"], state=ops["initial_state"])
    for b in (dict(state=torch.zeros(8, 2, device=DEV).t()), dict(state=row["state"].bfloat16()), dict(x=x[:, 0].bfloat16()), dict(x=x),
              dict(c=-1.0), dict(decay=ops["decay"].clone().requires_grad_(True)), dict(state=row["state"].clone().requires_grad_(True))):
        with pytest.raises(ValueError):
            gated_recurrence_step(**{**row, **b})
    with torch.no_grad():
        gated_recurrence_step(**{**row, "decay": ops["decay"].clone().requires_grad_(True)})
