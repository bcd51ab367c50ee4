"""The two widths of a pass over the chunks, 16 value columns to a workgroup as long as every such
tile has a CU of its own (256), else 32: the same results to the bit on both sides of the border, and
the oracle's (four fp32 sums of at most 192 terms, and bf16's half step)."""
import pytest
import torch
import torch.nn.functional as F

from oracle import delta_oracle as O

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("heads, V", [(64, 64), (65, 64), (20, 200), (128, 64)], ids=["256", "260", "280", "512"])
def test_both_sides_of_the_border(heads, V):
    from gruboros_amd.delta import gated_delta_rule

    gen = torch.Generator().manual_seed(heads)
    T, K = 131, 24
    q, k = (F.normalize(F.silu(torch.randn(1, T, heads, K, generator=gen)), dim=-1) for _ in range(2))
    xs = [q, k, torch.randn(1, T, heads, V, generator=gen), -torch.rand(1, T, heads, generator=gen), torch.rand(1, T, heads, generator=gen)]
    xs, do = [t.bfloat16() for t in xs], torch.randn(1, T, heads, V, generator=gen).bfloat16()

    def run(xs, do):
        leaves = [t.to(DEV).requires_grad_(True) for t in xs]
        o = gated_delta_rule(*leaves)
        return [o, *torch.autograd.grad(o, leaves, do.to(DEV))]

    whole, few = run(xs, do), run([t[:, :, -3:] for t in xs], do[:, :, -3:])
    for a, b in zip(whole, few):
        assert torch.equal(a[:, :, -3:], b)
    rs = [t[:, :, -3:].double().requires_grad_(True) for t in xs]
    ro, _ = O.gated_delta_rule(*rs)
    for a, b in zip(few, [ro, *torch.autograd.grad(ro, rs, do[:, :, -3:].double())]):
        assert float((a.detach().double().cpu() - b.detach()).norm() / b.detach().norm()) <= 2.0 ** -8 + 1e-4
