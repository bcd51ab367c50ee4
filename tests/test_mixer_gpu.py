"""The operators in a run, as a block of a language model uses them: norm of the residual stream,
a projection to q, k, v, gates, the gated delta rule, a projection back, dropout of the branch on
its way into the stream together with the next norm, and a dropped feed-forward branch; trained
forward and backward, and generated with token by token from a prompt's state.

Against the same block in float64 with the oracles (the rule token by token, Philox's own keep
mask). Tolerance: eight operators in a row, each within the delta rule's 5e-5 of its own terms
(float32: products of up to 1024 terms, 1024 2^-24 = 6e-5), and gradients through as many again:
16 * 6e-5 = 1e-3."""
import pytest
import torch
import torch.nn.functional as F

from oracle import delta_oracle as O
from oracle import philox

pytestmark = pytest.mark.gpu
DEV = "cuda"
TOL = 1e-3
B, T, D, HK, H, K, V, P = 2, 90, 96, 2, 4, 16, 24, 0.2


def _params():
    gen = torch.Generator().manual_seed(11)

    def normal(*s, scale=1.0):
        return scale * torch.randn(*s, generator=gen)

    n = 2 * HK * K + H * V + 2 * H
    return {"x": normal(B, T, D), "w1": 1 + normal(D, scale=0.1), "b1": normal(D, scale=0.1), "proj": normal(n, D, scale=D ** -0.5),
            "out": normal(D, H * V, scale=(H * V) ** -0.5), "w2": 1 + normal(D, scale=0.1), "b2": normal(D, scale=0.1),
            "up": normal(2 * D, D, scale=D ** -0.5), "down": normal(D, 2 * D, scale=(2 * D) ** -0.5)}, normal(B, T, D)


def _split(z):
    q, k, v, g, beta = z.split([HK * K, HK * K, H * V, H, H], -1)
    q, k = (F.normalize(t.unflatten(-1, (HK, K)), dim=-1) for t in (q, k))
    return q, k, v.unflatten(-1, (H, V)), -F.softplus(g), torch.sigmoid(beta)


def _block(p, seed):
    """The framework's operators."""
    from gruboros_amd.delta import gated_delta_rule
    from gruboros_amd.dropout import dropout
    from gruboros_amd.norm import add_layer_norm, layer_norm

    z = layer_norm(p["x"], p["w1"], p["b1"]) @ p["proj"].T
    o, state = gated_delta_rule(*_split(z), return_state=True)
    xn, y = add_layer_norm(p["x"], o.flatten(2) @ p["out"].T, p["w2"], p["b2"], dropout_p=P if seed is not None else 0.0, seed=seed, offset=1)
    ff = F.silu(y @ p["up"].T) @ p["down"].T
    return (dropout(ff, P, seed, offset=2, residual=xn) if seed is not None else xn + ff), state


def _double(p, seed):
    def norm(x, w, b):
        return F.layer_norm(x, (D,), w, b, 1e-5)

    def drop(x, offset):
        if seed is None:
            return x
        return x * torch.as_tensor(philox.keep(x.numel(), P, seed, offset)).view(x.shape) / (1 - P)

    o, state = O.gated_delta_rule(*_split(norm(p["x"], p["w1"], p["b1"]) @ p["proj"].T))
    xn = p["x"] + drop(o.flatten(2) @ p["out"].T, 1)
    ff = F.silu(norm(xn, p["w2"], p["b2"]) @ p["up"].T) @ p["down"].T
    return xn + drop(ff, 2), state


def _off(a, b):
    b = b.detach().double()
    return float((a.detach().double().cpu() - b).norm() / b.norm())


def test_training_step():
    p, dy = _params()
    ours = {n: t.to(DEV).requires_grad_(True) for n, t in p.items()}
    ref = {n: t.double().requires_grad_(True) for n, t in p.items()}
    y, _ = _block(ours, 1234)
    ry, _ = _double(ref, 1234)
    assert _off(y, ry) <= TOL
    got = torch.autograd.grad(y, list(ours.values()), dy.to(DEV))
    want = torch.autograd.grad(ry, list(ref.values()), dy.double())
    for n, a, b in zip(p, got, want):
        assert _off(a, b) <= TOL, n


def test_recomputed_branch_drops_the_same():
    """Under torch's checkpointing the block runs again in the backward, and drops the same values."""
    from torch.utils.checkpoint import checkpoint

    p, dy = _params()
    ours = {n: t.to(DEV).requires_grad_(True) for n, t in p.items()}
    want = torch.autograd.grad(_block(ours, 77)[0], list(ours.values()), dy.to(DEV))
    y = checkpoint(lambda *a: _block(dict(zip(p, a)), 77)[0], *ours.values(), use_reentrant=False)
    got = torch.autograd.grad(y, list(ours.values()), dy.to(DEV))
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_generation():
    """A prompt of 80 tokens, then ten by single steps, against the whole sequence at once."""
    from gruboros_amd.delta import gated_delta_step
    from gruboros_amd.norm import add_layer_norm, layer_norm

    p, _ = _params()
    ry, rs = _double({n: t.double() for n, t in p.items()}, None)
    p = {n: t.to(DEV) for n, t in p.items()}
    with torch.no_grad():
        y, state = _block({**p, "x": p["x"][:, :80]}, None)
        assert _off(y, ry[:, :80]) <= TOL
        for t in range(80, T):
            x = p["x"][:, t]
            o = gated_delta_step(*_split(layer_norm(x, p["w1"], p["b1"]) @ p["proj"].T), state)
            xn, z = add_layer_norm(x, o.flatten(1) @ p["out"].T, p["w2"], p["b2"])
            assert _off(xn + F.silu(z @ p["up"].T) @ p["down"].T, ry[:, t]) <= TOL
    assert _off(state, rs) <= TOL
