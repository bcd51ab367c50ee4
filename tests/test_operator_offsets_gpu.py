"""Operands of more than 2^31 values (dropout: 2^32): offsets that 32 bits do not hold. The last rows
are those of a short call on them alone, to the bit, and dropout's words those of their index."""
import pytest
import torch

from oracle import philox

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.fixture(autouse=True)
def _memory():
    yield
    torch.cuda.empty_cache()  # (120 GB that no other test needs)


def test_delta_rule():
    """64 heads over 262344 tokens. At token 262144, a chunk's first, all is forgotten: from there on,
    outputs and gradients are those of a sequence that begins there."""
    from gruboros_amd.delta import gated_delta_rule

    H, K, V, at = 64, 128, 128, 262144
    T = at + 200
    gen = torch.Generator(device=DEV).manual_seed(8)

    def normal(*s):
        return torch.randn(*s, generator=gen, device=DEV, dtype=torch.bfloat16)

    xs = [normal(1, T, H, K).mul_(K ** -0.5), normal(1, T, H, K).mul_(K ** -0.5), normal(1, T, H, V), normal(1, T, H).abs_().neg_(),
          torch.sigmoid(normal(1, T, H))]
    xs[3][:, at] = -float("inf")
    do = normal(1, T, H, V)
    assert xs[0].numel() > 1 << 31

    def run(place):
        leaves = [place(t).requires_grad_(True) for t in xs]
        o, s = gated_delta_rule(*leaves, return_state=True)
        return [o, s, *torch.autograd.grad(o, leaves, place(do))]

    short = run(lambda t: t[:, at:].clone())
    long = run(lambda t: t)
    for a, b in zip(long, short):
        assert bool(b.isfinite().all()) and torch.equal(a if a.dim() == 4 and a.shape[1] == H else a[:, at:], b)


def test_layer_norm():
    from gruboros_amd.norm import layer_norm

    N, D = (1 << 21) + 3, 1024
    gen = torch.Generator(device=DEV).manual_seed(9)
    x, dy = (torch.randn(N, D, generator=gen, device=DEV, dtype=torch.bfloat16) for _ in range(2))
    w = torch.randn(D, generator=gen, device=DEV)

    def run(x, dy):
        x = x.requires_grad_(True)
        y = layer_norm(x, w)
        return y, torch.autograd.grad(y, x, dy)[0]

    for a, b in zip(run(x, dy), run(x.detach()[-5:].clone(), dy[-5:])):
        assert torch.equal(a[-5:], b)


def test_dropout():
    from gruboros_amd.dropout import dropout

    n, p, seed, offset = (1 << 32) + 37, 0.5, (1 << 60) + 5, (1 << 40) + 1
    y = dropout(torch.ones(n, device=DEV, dtype=torch.bfloat16), p, seed, offset=offset)
    for first in ((1 << 31) - 20, (1 << 32) - 20):
        want = torch.from_numpy(philox.words(57, seed, offset, first) >= int(p * 2 ** 32))
        assert torch.equal(y[first:first + 57].cpu() != 0, want)
    del y
    # the branch of a norm draws the same words
    from gruboros_amd.norm import add_layer_norm

    N, D = (1 << 21) + 3, 1024
    x, d = torch.zeros(N, D, device=DEV), torch.ones(N, D, device=DEV, dtype=torch.bfloat16)
    xn, _ = add_layer_norm(x, d, torch.ones(D, device=DEV), out_dtype=torch.bfloat16, dropout_p=p, seed=seed, offset=offset)
    want = torch.from_numpy(philox.words(3 * D, seed, offset, (N - 3) * D) >= int(p * 2 ** 32)).view(3, D)
    assert torch.equal(xn[-3:].cpu() != 0, want)
