"""Batches and sequences of no values, trained on: a backward pass gives every operand a gradient of
zeros (torch's own operators do), the weights of a norm among them, instead of finding no graph."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
TYPES = pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])


def _zeros(outs, leaves):
    grads = torch.autograd.grad([o.sum() for o in outs], leaves)
    assert all(g.shape == t.shape and g.dtype == t.dtype and bool((g == 0).all()) for g, t in zip(grads, leaves))


def _leaves(*tensors):
    return [t.to(DEV).requires_grad_(True) for t in tensors]


@TYPES
@pytest.mark.parametrize("size", [(0, 5), (2, 0), (0, 0)], ids=str)
def test_rule(size, dtype):
    from gruboros_amd.delta import gated_delta_rule

    (B, T), n = size, torch.zeros
    leaves = _leaves(n(B, T, 1, 16, dtype=dtype), n(B, T, 1, 16, dtype=dtype), n(B, T, 2, 8, dtype=dtype), n(B, T, 2, dtype=dtype),
                     n(B, T, 2, dtype=dtype))
    _zeros([gated_delta_rule(*leaves)], leaves)
    (h0,) = _leaves(torch.full((B, 2, 16, 8), float("inf")))  # (its values are not what the zeros come from)
    o = gated_delta_rule(*leaves, initial_state=h0)
    assert o.dtype == dtype and o.shape == leaves[2].shape
    _zeros([o], [*leaves, h0])
    o, s = gated_delta_rule(*leaves, initial_state=h0, return_state=True)
    assert torch.equal(torch.autograd.grad([o.sum(), s.sum()], h0)[0], torch.ones_like(h0)) and torch.equal(s, h0)
    if B == 0:
        _zeros([gated_delta_rule(*leaves, return_state=True)[1]], [leaves[1], leaves[2], leaves[3], leaves[4]])


@TYPES
def test_norms(dtype):
    from gruboros_amd.norm import add_layer_norm, layer_norm

    leaves = _leaves(torch.zeros(0, 3, 16, dtype=dtype), torch.ones(16, dtype=dtype), torch.ones(16))
    y = layer_norm(*leaves)
    assert y.dtype == dtype
    _zeros([y], leaves)
    _zeros([layer_norm(*leaves[:2])], leaves[:2])
    leaves = _leaves(torch.zeros(0, 16), torch.zeros(0, 16, dtype=dtype), torch.ones(16), torch.ones(16))
    xn, y = add_layer_norm(*leaves, out_dtype=dtype)
    assert y.dtype == dtype
    _zeros([y], leaves)
    _zeros([xn], leaves[:2])


@TYPES
def test_dropout(dtype):
    from gruboros_amd.dropout import dropout

    leaves = _leaves(torch.zeros(0, 4, dtype=dtype), torch.zeros(0, 4))
    _zeros([dropout(leaves[0], 0.5, 1)], leaves[:1])
    _zeros([dropout(leaves[0], 0.5, 1, residual=leaves[1])], leaves)
