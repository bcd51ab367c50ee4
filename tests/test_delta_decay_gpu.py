"""The gradient of the decay, head by head and token by token, from heads that forget little to heads
that forget nearly all: relative to itself, as an optimiser sees it that normalises it.

With A = e^g S the decayed state and A' the loss's gradient by it, dg = sum over K x V of A A'. Its
terms cannot be better than what A and A' are made of: sums of at most n = 768 terms in fp32 one after
the other, each partial sum off by half a step, 2^-24 of sqrt(n) terms' size if the terms' signs are
mixed, so that n roundings make n 2^-24 = 4.6e-5 of the sum's own size, sqrt(n) terms: F32 = 5e-5 of
the root of the terms' squares. bfloat16 adds half a step of dg, 2^-8, and two roundings to 2^-17 of
what the backward keeps, within the 1e-4 that it has in place of F32."""
import pytest
import torch
import torch.nn.functional as F

pytestmark = pytest.mark.gpu
DEV = "cuda"
TYPES = pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
DECAYS = [-0.01, -0.3, -1.0, -4.0, -8.0, -12.0, -20.0, -40.0]


def _inputs(B, T, Hk, H, K, V, dtype):
    gen = torch.Generator().manual_seed(11 * T + K)
    q, k = (F.normalize(F.silu(torch.randn(B, T, Hk, K, generator=gen)), dim=-1) for _ in range(2))
    v, beta = torch.randn(B, T, H, V, generator=gen), torch.sigmoid(torch.randn(B, T, H, generator=gen))
    more = [torch.randn(B, H, K, V, generator=gen) for _ in range(2)]
    return [t.to(dtype) for t in (q, k, v, beta)], torch.randn(B, T, H, V, generator=gen).to(dtype), *more


def _reference(q, k, v, g, beta, h0, do, ds):
    """dg [B, T, H] in float64, token by token, and the root of its terms' squares."""
    q, k, v, g, beta, h0, do, ds = (t.double() for t in (q, k, v, g, beta, h0, do, ds))
    q, k = (t.repeat_interleave(v.shape[2] // t.shape[2], 2) for t in (q, k))
    S, seen, out = h0, [], []
    for t in range(v.shape[1]):
        A = (g[:, t].exp()[..., None, None] * S).detach().requires_grad_(True)
        seen.append(A)
        err = v[:, t] - (k[:, t].unsqueeze(-1) * A).sum(-2)
        S = A + (beta[:, t].unsqueeze(-1) * k[:, t]).unsqueeze(-1) * err.unsqueeze(-2)
        out.append((S, (q[:, t].unsqueeze(-1) * S).sum(-2) * q.shape[-1] ** -0.5))
    dg, size, dS = [], [], ds
    for t in reversed(range(v.shape[1])):  # (each token's graph by itself: A is a leaf)
        (dA,) = torch.autograd.grad(out[t], seen[t], [dS, do[:, t]])
        terms = (dA * seen[t]).detach().flatten(2)
        dg.append(terms.sum(-1))
        size.append(terms.square().sum(-1).sqrt())
        dS = g[:, t].exp()[..., None, None] * dA
    return torch.stack(dg[::-1], 1), torch.stack(size[::-1], 1)


def _dg(q, k, v, g, beta, h0, do, ds):
    from gruboros_amd.delta import gated_delta_rule

    q, k, v, g, beta, h0, do, ds = (t.to(DEV) for t in (q, k, v, g, beta, h0, do, ds))
    g.requires_grad_(True)
    o, s = gated_delta_rule(q, k, v, g, beta, initial_state=h0, return_state=True)
    return torch.autograd.grad([o, s], g, [do, ds])[0].double().cpu()


def _limit(dtype, dg, size):
    return 5e-5 * size if dtype == torch.float32 else 2.0 ** -8 * dg + 1e-4 * size


@TYPES
@pytest.mark.parametrize("sizes", [(2, 64, 32), (8, 64, 64), (4, 128, 128), (8, 40, 24)], ids=str)
def test_every_head_by_itself(sizes, dtype):
    """One decay per head, as slow and fast heads have them."""
    Hk, K, V = sizes
    (q, k, v, beta), do, h0, ds = _inputs(2, 131, Hk, len(DECAYS), K, V, dtype)
    jitter = torch.rand(2, 131, len(DECAYS), generator=torch.Generator().manual_seed(1))
    g = (torch.tensor(DECAYS) * (0.9 + 0.2 * jitter)).to(dtype)
    got = _dg(q, k, v, g, beta, h0, do, ds)
    want, size = _reference(q, k, v, g, beta, h0, do, ds)
    off = (got - want).norm(dim=(0, 1)) / _limit(dtype, want.norm(dim=(0, 1)), size.norm(dim=(0, 1)))
    print([f"{x:.2f}" for x in off.tolist()])
    assert bool((off <= 1).all()), off


@TYPES
def test_single_tokens_that_forget(dtype):
    """A head that forgets little, and nearly all at a few tokens: those tokens' own gradients, beside
    neighbours 10^4 to 10^17 times as large."""
    (q, k, v, beta), do, h0, ds = _inputs(2, 131, 2, 4, 64, 32, dtype)
    g = torch.full((2, 131, 4), -0.05)
    at = [0, 1, 17, 40, 63, 64, 100, 130]
    for h, d in enumerate((-10.0, -16.0, -24.0, -40.0)):
        g[:, at, h] = d
    g = g.to(dtype)
    got = _dg(q, k, v, g, beta, h0, do, ds)
    want, size = _reference(q, k, v, g, beta, h0, do, ds)
    off = (got - want).abs() / _limit(dtype, want.abs(), size)
    print(f"worst {float(off[:, at].max()):.2f} at those tokens, {float(off.max()):.2f} at all")
    assert bool((off <= 1).all())
