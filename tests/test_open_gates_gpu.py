"""Gradients of gates that are far open or far shut, value by value: they are those of 1 - sigmoid(g), which a
difference from 1 has lost by then.

Tolerance before any run: a sigmoid and its complement at |g| <= 20 are a power of two whose argument is rounded twice
at 20 log2(e) = 29 (29 ln 2 2^-23 = 2.4e-6), 1 + e, a reciprocal and a product: 3e-6 each; a gradient has at most
three such factors and the decay's terms, which are as near: 1e-5 of its value. The operands leave no difference in it.
"""
import pytest
import torch

from oracle.recurrence_oracle import gated_recurrence as oracle

pytestmark = pytest.mark.gpu
DEV = "cuda"
f32, bf16 = torch.float32, torch.bfloat16
GATES = torch.tensor([-20.0, -16.0, -10.0, -4.0, -1.0, 0.0, 1.0, 4.0, 10.0, 14.0, 16.0, 18.0, 20.0])
LIMIT = 1e-5


def _near(got, want, what):
    half = 2.0 ** -8 if got.dtype == bf16 else 0.0
    err = (got.double().cpu() - want).abs()
    assert bool((err <= (LIMIT + half) * want.abs()).all()), f"{what}: {float((err / want.abs()).max()):.2e}"


@pytest.mark.parametrize("dtype", [f32, bf16], ids=["f32", "bf16"])
def test_recurrence(dtype):
    """One token: negative x on a positive state, so that both parts of the decay's gradient have one sign."""
    from gruboros_amd.recurrence import gated_recurrence

    n = len(GATES)
    gen = torch.Generator().manual_seed(0)
    draw = lambda *s: 0.5 + torch.rand(*s, generator=gen)  # noqa: E731
    for decay in (-8.0, -3.0, 0.0):
        ops = [-draw(n, 1, n).to(dtype), GATES.view(n, 1, 1).expand(n, 1, n).to(dtype), GATES.expand(n, 1, n).to(dtype), torch.full((n,), decay),
               draw(n, n)]
        dh = draw(n, 1, n).to(dtype)
        ref = [t.double().requires_grad_(True) for t in ops]
        want = torch.autograd.grad(oracle(*ref)[0], ref, dh.double())
        dev = [t.to(DEV).requires_grad_(True) for t in ops]
        got = torch.autograd.grad(gated_recurrence(*dev), dev, dh.to(DEV))
        for name, g, w in zip(("x", "input_gate", "decay_gate", "decay", "initial_state"), got, want):
            _near(g, w, f"d{name}, decay {decay}")


@pytest.mark.parametrize("dtype", [f32, bf16], ids=["f32", "bf16"])
@pytest.mark.parametrize("activation", ["sigmoid", "silu"])
def test_block_norm(activation, dtype):
    from gruboros_amd.norm import add_gated_rms_norm

    n = len(GATES)
    gen = torch.Generator().manual_seed(1)
    x, branch, dres = (0.5 + torch.rand(n, n, generator=gen) for _ in range(3))
    branch, gate, w = branch.to(dtype), GATES.expand(n, n).to(dtype).contiguous(), torch.ones(n)
    ref = gate.double().requires_grad_(True)
    f = branch.double()
    b = f / (f.square().mean(-1, keepdim=True) + 1e-6).sqrt() * torch.sigmoid(ref) * (ref if activation == "silu" else 1.0)
    (want,) = torch.autograd.grad(b, ref, dres.double())
    leaf = gate.to(DEV).requires_grad_(True)
    xn, _ = add_gated_rms_norm(x.to(DEV), branch.to(DEV), w.to(DEV), w.to(DEV), gate=leaf, activation=activation, eps=1e-6)
    _near(torch.autograd.grad(xn, leaf, dres.to(DEV))[0], want, "dgate")
