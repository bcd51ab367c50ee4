"""Calls of the gated delta rule that a program makes beside the plain one: views of a packed
projection, broadcast operands, decays that forget all, empty batches, another stream, captured
steps, the two widths of a pass over the chunks, large states; and what it refuses.

The oracle is the rule token by token in float64; tolerances are those of the parity tests there
(4 sums of at most 192 terms in fp32: 5e-5; bf16's half step 2^-8 besides)."""
import pytest
import torch
import torch.nn.functional as F

from oracle import delta_oracle as O

pytestmark = pytest.mark.gpu
DEV = "cuda"
F32, BF16 = 5e-5, 2.0 ** -8 + 1e-4
NAMES = ("q", "k", "v", "g", "beta")


def _inputs(B, T, Hk, H, K, V, dtype=torch.float32, seed=0):
    gen = torch.Generator().manual_seed(seed + 7 * T + K)
    q, k = (F.normalize(F.silu(torch.randn(B, T, Hk, K, generator=gen)), dim=-1) for _ in range(2))
    x = [q, k, torch.randn(B, T, H, V, generator=gen), -0.3 * F.softplus(torch.randn(B, T, H, generator=gen)),
         torch.sigmoid(torch.randn(B, T, H, generator=gen))]
    return [t.to(dtype) for t in x], torch.randn(B, T, H, V, generator=gen).to(dtype)


def _off(a, b):
    b = b.detach().double().cpu()
    return float((a.detach().double().cpu() - b).norm() / b.norm().clamp_min(1e-30))


def _double(xs):
    return [t.detach().double().cpu().requires_grad_(True) for t in xs]


def test_views_of_a_packed_projection():
    """q, k, v as slices of one [B, T, (2 Hk K + H V)] tensor, g and beta of another; the gradient of
    the packed tensors, and a do that is a slice too."""
    from gruboros_amd.delta import gated_delta_rule

    B, T, Hk, H, K, V = 2, 130, 2, 4, 64, 32
    (q, k, v, g, beta), do = _inputs(B, T, Hk, H, K, V)
    packed = torch.cat([t.flatten(2) for t in (q, k, v)], -1)
    gates = torch.cat([g, beta], -1)

    def split(p, e):
        a, b, c = p.split([Hk * K, Hk * K, H * V], -1)
        return (a.unflatten(-1, (Hk, K)), b.unflatten(-1, (Hk, K)), c.unflatten(-1, (H, V)), *e.split([H, H], -1))

    wide = torch.zeros(B, T, H, V + 8, device=DEV)
    wide[..., :V] = do.to(DEV)
    p, e = packed.to(DEV).requires_grad_(True), gates.to(DEV).requires_grad_(True)
    o = gated_delta_rule(*split(p, e))
    got = torch.autograd.grad(o, (p, e), wide[..., :V])
    rp, re = _double((packed, gates))
    ro, _ = O.gated_delta_rule(*split(rp, re))
    want = torch.autograd.grad(ro, (rp, re), do.double())
    assert _off(o, ro) <= F32 and _off(got[0], want[0]) <= F32
    # (dg is a difference of terms about as large as dq . q: eight times the tolerance of a sum)
    assert _off(got[1], want[1]) <= 8 * F32


def test_rows_at_odd_places():
    """Operands whose rows are not at multiples of 16 bytes, a transposed batch and head-major storage."""
    from gruboros_amd.delta import gated_delta_rule

    xs, _ = _inputs(2, 70, 2, 2, 40, 24)
    want = gated_delta_rule(*(t.to(DEV) for t in xs))

    def odd(t):
        buf = torch.zeros(t.numel() + 1, device=DEV)
        buf[1:] = t.flatten().to(DEV)
        return buf[1:].view(t.shape)

    def head_major(t):
        return t.to(DEV).transpose(1, 2).contiguous().transpose(1, 2)

    def wide(t):  # inner rows of 41 values
        buf = torch.zeros(*t.shape[:-1], t.shape[-1] + 1, device=DEV)
        buf[..., :-1] = t.to(DEV)
        return buf[..., :-1]

    for f in (odd, head_major, wide):
        assert torch.equal(gated_delta_rule(*(f(t) for t in xs)), want)


def test_broadcast_operands():
    """One beta for all tokens, one v for the batch: their gradients are sums."""
    from gruboros_amd.delta import gated_delta_rule

    (q, k, v, g, beta), do = _inputs(3, 70, 1, 2, 16, 8)

    def f(rule, q, k, v1, g, b1):
        out = rule(q, k, v1.expand(3, -1, -1, -1), g, b1.expand(3, 70, 2))
        return out[0] if isinstance(out, tuple) else out

    small = [q, k, v[:1], g, beta[:1, :1]]
    xs, rs = [t.to(DEV).requires_grad_(True) for t in small], _double(small)
    o, ro = f(gated_delta_rule, *xs), f(O.gated_delta_rule, *rs)
    got, want = torch.autograd.grad(o, xs, do.to(DEV)), torch.autograd.grad(ro, rs, do.double())
    assert _off(o, ro) <= F32
    for a, b in zip(got, want):
        assert a.shape == b.shape and _off(a, b) <= 8 * F32


@pytest.mark.parametrize("at", [0, 1, 63, 64, 69])
def test_forgetting(at):
    """g = -inf: the outputs from there on are those of a sequence that begins there; its gradients too,
    and nothing reaches what was forgotten."""
    from gruboros_amd.delta import gated_delta_rule

    (q, k, v, g, beta), do = _inputs(1, 70, 1, 2, 32, 16)
    g[:, at] = -float("inf")
    xs = [t.to(DEV).requires_grad_(True) for t in (q, k, v, g, beta)]
    h0 = torch.ones(1, 2, 32, 16, device=DEV, requires_grad=True)
    o, s = gated_delta_rule(*xs, initial_state=h0, return_state=True)
    tail = do.to(DEV).clone()
    tail[:, :at] = 0
    grads = torch.autograd.grad([o, s], [*xs, h0], [tail, torch.ones_like(s)])
    rs = _double([t[:, at:] for t in (q, k, v, g.clamp_min(-500.0), beta)])  # (e^-500 is 0 beside anything here)
    ro, rstate = O.gated_delta_rule(*rs)
    want = torch.autograd.grad([ro, rstate], rs, [do[:, at:].double(), torch.ones_like(rstate)])
    assert _off(o[:, at:], ro) <= F32 and _off(s, rstate) <= F32
    for a, b in zip(grads[:5], want):
        assert a.isfinite().all() and _off(a[:, at:], b) <= 8 * F32
        assert at == 0 or float(a[:, :at].abs().max()) <= 1e-6
    assert float(grads[5].abs().max()) <= 1e-30


def test_nothing_written_and_no_decay():
    """beta = 0: the state only decays. g = 0, beta = 1: the delta rule without gates."""
    from gruboros_amd.delta import gated_delta_rule

    (q, k, v, g, beta), _ = _inputs(1, 100, 1, 1, 24, 16)
    h0 = torch.randn(1, 1, 24, 16, generator=torch.Generator().manual_seed(3))
    for gg, bb in ((g, torch.zeros_like(beta)), (torch.zeros_like(g), torch.ones_like(beta))):
        o, s = gated_delta_rule(*(t.to(DEV) for t in (q, k, v, gg, bb)), initial_state=h0.to(DEV), return_state=True)
        ro, rs = O.gated_delta_rule(*(t.double() for t in (q, k, v, gg, bb, h0)))
        assert _off(o, ro) <= F32 and _off(s, rs) <= F32


def test_no_tokens():
    from gruboros_amd.delta import gated_delta_rule, gated_delta_step

    for B, T in ((0, 5), (2, 0)):
        q, v, g = torch.zeros(B, T, 1, 16, device=DEV), torch.zeros(B, T, 2, 8, device=DEV), torch.zeros(B, T, 2, device=DEV)
        h0 = torch.ones(B, 2, 16, 8, device=DEV)
        o, s = gated_delta_rule(q, q, v, g, g, initial_state=h0, return_state=True)
        assert o.shape == v.shape and torch.equal(s, h0)
        assert gated_delta_rule(q, q, v, g, g).shape == v.shape
    e = torch.zeros(0, 1, 16, device=DEV)
    assert gated_delta_step(e, e, e, e[..., 0], e[..., 0], torch.zeros(0, 1, 16, 16, device=DEV)).shape == e.shape


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("T", [64, 200])
def test_enough_heads_for_two_tiles(T, dtype):
    """64 heads of 128 value columns: a workgroup of a pass takes 32 columns (bf16), against 16 with fewer
    heads. Both give the same results, to the bit."""
    from gruboros_amd.delta import gated_delta_rule

    xs, do = _inputs(4, T, 16, 16, 32, 128, dtype)
    dev = [t.to(DEV).requires_grad_(True) for t in xs]
    o = gated_delta_rule(*dev)
    grads = torch.autograd.grad(o, dev, do.to(DEV))
    one = [t[:1].to(DEV).requires_grad_(True) for t in xs]
    o1 = gated_delta_rule(*one)
    g1 = torch.autograd.grad(o1, one, do[:1].to(DEV))
    assert torch.equal(o[:1], o1) and all(torch.equal(a[:1], b) for a, b in zip(grads, g1))
    ro, _ = O.gated_delta_rule(*(t[3:, :, 14:].double() for t in xs))
    assert _off(o[3:, :, 14:], ro) <= (F32 if dtype == torch.float32 else BF16)


def test_gradients_against_differences():
    """Along random directions, central differences of the kernels' own fp32 forward. With a step of 2^-6
    the difference's error is of third order in it (2^-12 of the curvature's size) and 2^-24 2^6 of the
    loss's terms from rounding: 2e-3 together covers both with a margin of 4."""
    from gruboros_amd.delta import gated_delta_rule

    xs, do = _inputs(1, 67, 1, 2, 16, 8, seed=5)
    gen = torch.Generator().manual_seed(9)
    xs, do = [t.to(DEV) for t in (*xs, torch.randn(1, 2, 16, 8, generator=gen))], do.to(DEV)
    leaves = [t.clone().requires_grad_(True) for t in xs]
    grads = torch.autograd.grad(gated_delta_rule(*leaves[:5], initial_state=leaves[5]), leaves, do)

    def loss(ts):
        return float((gated_delta_rule(*ts[:5], initial_state=ts[5]).double() * do.double()).sum())

    h = 2.0 ** -6
    for i, t in enumerate(xs):
        d = torch.randn(t.shape, generator=gen).to(DEV)
        d /= d.norm()
        up, down = ([u + s * h * d if j == i else u for j, u in enumerate(xs)] for s in (1, -1))
        want = (loss(up) - loss(down)) / (2 * h)
        assert abs(float((grads[i].double() * d).sum()) - want) <= 2e-3 * max(1.0, float(grads[i].norm())), i


def test_another_stream():
    """Operands made on one stream, the rule run on another that waits for it."""
    from gruboros_amd.delta import gated_delta_rule, gated_delta_step

    xs, do = _inputs(2, 300, 2, 2, 64, 64, torch.bfloat16)
    dev = [t.to(DEV).requires_grad_(True) for t in xs]
    dod = do.to(DEV)

    def work():
        o, s = gated_delta_rule(*dev, return_state=True)
        out = [o, s, *torch.autograd.grad(o, dev, dod)]
        with torch.no_grad():
            s2 = s.clone()
            out += [gated_delta_step(*(t[:, 0] for t in dev), s2), s2]
        return out

    want = work()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = work()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_captured_step_and_backward():
    """A training pass and a generated token in two graphs, replayed in turn with eager work in between."""
    from gruboros_amd.delta import gated_delta_rule, gated_delta_step

    xs, do = _inputs(2, 150, 1, 2, 64, 32)
    dev = [t.to(DEV) for t in xs]
    dod = do.to(DEV)
    state = torch.zeros(2, 2, 64, 32, device=DEV)
    tok = [t[:, 0].clone() for t in dev]

    def train():
        leaves = [t.detach().requires_grad_(True) for t in dev]
        o = gated_delta_rule(*leaves)
        return [o.detach(), *torch.autograd.grad(o, leaves, dod)]

    def token():
        return gated_delta_step(*tok, state)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        train(), token()
    torch.cuda.current_stream().wait_stream(side)
    g1, g2 = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(g1):
        out = train()
    with torch.cuda.graph(g2):
        o2 = token()
    for i in range(3):
        for t in dev:
            t.mul_(0.9)
        for t in tok:
            t.mul_(0.9)
        state.fill_(0.5)
        g1.replay()
        g2.replay()
        torch.cuda.synchronize()
        got, gs = [t.clone() for t in (*out, o2)], state.clone()
        want = train()
        state.fill_(0.5)
        want.append(token())
        assert all(torch.equal(a, b) for a, b in zip(got, want)) and torch.equal(gs, state)


@pytest.mark.parametrize("B", [1, 64], ids=["8 MiB at most", "64 MiB"])
def test_step_of_large_states(B):
    """From 64 MiB on a step goes past the caches: the same results, and only its own state is written."""
    from gruboros_amd.delta import gated_delta_step

    H, K, V = 16, 128, 128
    gen = torch.Generator().manual_seed(2)
    x = [torch.randn(B, H, n, generator=gen).to(DEV) / n ** 0.5 for n in (K, K, V)]
    g, beta = -torch.rand(B, H, generator=gen).to(DEV), torch.rand(B, H, generator=gen).to(DEV)
    room = torch.full((B + 2, H, K, V), 3.0, device=DEV)
    state = room[1:-1]
    state.copy_(torch.randn(H, K, V, generator=gen).to(DEV).expand(B, H, K, V))
    s = state.double() * g.double().exp()[..., None, None]
    q, k, v = (t.double() for t in x)
    d = beta.double()[..., None] * (v - (k.unsqueeze(-1) * s).sum(-2))
    s += k.unsqueeze(-1) * d.unsqueeze(-2)
    o = gated_delta_step(*x, g, beta, state)
    assert _off(o, K ** -0.5 * (q.unsqueeze(-1) * s).sum(-2)) <= F32 and _off(state, s) <= F32
    assert bool((room[0] == 3).all()) and bool((room[-1] == 3).all())


def test_refusals():
    from gruboros_amd._lib import MingruHipError
    from gruboros_amd.delta import gated_delta_rule, gated_delta_step

    (q, k, v, g, beta), _ = _inputs(2, 10, 2, 4, 16, 8)
    x = [t.to(DEV) for t in (q, k, v, g, beta)]
    q, k, v, g, beta = x

    def bad(error, *args, **kw):
        with pytest.raises(error):
            gated_delta_rule(*args, **kw)

    bad(ValueError, q, k[:, :9], v, g, beta)
    bad(ValueError, q, k, v[:, :9], g, beta)
    bad(ValueError, q, k, v[:, :, :3], g[..., :3], beta[..., :3])  # 3 value heads on 2
    bad(ValueError, q[..., :12], k[..., :12], v, g, beta)
    bad(ValueError, q, k, v[..., :4], g, beta)
    bad(ValueError, q, k, v, g[..., :1], beta)
    bad(ValueError, q, k, v, g.bfloat16(), beta)
    bad(MingruHipError, *(t.half() for t in x))
    bad(ValueError, *x, initial_state=torch.zeros(2, 4, 8, 16, device=DEV))
    bad(ValueError, *x, initial_state=torch.zeros(2, 4, 16, 8, device=DEV).bfloat16())
    bad(MingruHipError, *x, initial_state=torch.zeros(2, 4, 16, 8))
    bad(ValueError, q[0], k[0], v[0], g[0], beta[0])
    tok, state = [t[:, 0] for t in x], torch.zeros(2, 4, 16, 8, device=DEV)
    with pytest.raises(ValueError):
        gated_delta_step(*tok, state.transpose(0, 1).contiguous().transpose(0, 1))
    with pytest.raises(ValueError):
        gated_delta_step(tok[0].clone().requires_grad_(True), *tok[1:], state)
    with pytest.raises(ValueError):
        gated_delta_step(*tok, state.bfloat16())


def test_one_derivative_only():
    from gruboros_amd.delta import gated_delta_rule, gated_delta_step

    xs, _ = _inputs(1, 5, 1, 1, 8, 8)
    xs = [t.to(DEV).requires_grad_(True) for t in xs]
    (g,) = torch.autograd.grad(gated_delta_rule(*xs).sum(), xs[2], create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()
    # an operand changed between the passes, or a state that a later step has moved on, is an error
    o = gated_delta_rule(*xs)
    with torch.no_grad():
        xs[0].add_(1.0)
    with pytest.raises(RuntimeError):
        o.sum().backward()
    state = torch.zeros(1, 1, 8, 8, device=DEV)
    w = torch.ones(1, 1, 8, 8, device=DEV, requires_grad=True)
    y = (w * state).sum()
    with torch.no_grad():
        gated_delta_step(*(t[:, 0] for t in xs), state)
    with pytest.raises(RuntimeError):
        y.backward()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("T", [1, 70])
def test_the_first_decay_without_a_state(T, dtype):
    """Nothing is there to decay at the first token: its g has no gradient at all, exactly."""
    from gruboros_amd.delta import gated_delta_rule

    xs, do = _inputs(2, T, 1, 2, 72, 40, dtype)
    dev = [t.to(DEV).requires_grad_(True) for t in xs]
    for h0 in (None, torch.zeros(2, 2, 72, 40, device=DEV)):
        dg = torch.autograd.grad(gated_delta_rule(*dev, initial_state=h0), dev, do.to(DEV))[3]
        assert bool((dg[:, 0] == 0).all()) and (T == 1 or bool((dg[:, 1:] != 0).any()))
    h0[1] = 1.0  # one sequence has a state
    dg = torch.autograd.grad(gated_delta_rule(*dev, initial_state=h0), dev, do.to(DEV))[3]
    assert bool((dg[0, 0] == 0).all()) and bool((dg[1, 0] != 0).all())
