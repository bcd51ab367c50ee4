"""What the bf16 rule's products see of an fp32 state: limbs that are rounded to nearest, off by 2^-18
at most and to either side. Cut limbs would be off by half of 2^-15 on average, always towards zero.

A chunk that writes nothing (beta = 0, g = 0) gives o = scale q S and dq = scale do S^T of its entry
state alone. Along the exact result the error is its bias: of N values rounded to bf16 the rounding,
to either side and of 2^-8 / sqrt(3) at most, leaves 2^-8 / sqrt(N) (normal values: sum x^4 = 3 N,
sum x^2 = N), 1.9e-6 for N = 2^22, and the slope of the values' density within a binade
2^-18 = 3.8e-6 at most. The limit 2^-17 = 7.6e-6 is more than both; limbs cut at 2^-15 lie
0.69 2^-16 = 1.05e-5 off (the mean of the cut part over mantissas from 1 to 2)."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"


def test_limbs_of_the_state_have_no_bias():
    from gruboros_amd.delta import gated_delta_rule

    B, T, H, K, V = 128, 64, 8, 64, 128
    gen = torch.Generator(device=DEV).manual_seed(4)

    def normal(*s):
        return torch.randn(*s, generator=gen, device=DEV)

    q, k, v, do = (normal(B, T, H, n).bfloat16() for n in (K, K, V, V))
    zero, h0 = torch.zeros(B, T, H, device=DEV, dtype=torch.bfloat16), normal(B, H, K, V)
    q.requires_grad_(True)
    o = gated_delta_rule(q, k, v, zero, zero, initial_state=h0, scale=1.0)
    (dq,) = torch.autograd.grad(o, q, do)
    S = h0.double()
    heads_first = [t.detach().double().transpose(1, 2).contiguous() for t in (q, do, o, dq)]
    want_o, want_dq = heads_first[0] @ S, heads_first[1] @ S.transpose(2, 3).contiguous()
    for name, got, want in (("o", heads_first[2], want_o), ("dq", heads_first[3], want_dq)):
        bias = float(((got - want) * want).sum() / want.square().sum())
        print(f"{name}: {bias:.2e}")
        assert abs(bias) <= 2.0 ** -17, name
