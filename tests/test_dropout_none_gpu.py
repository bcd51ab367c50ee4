"""Dropout with p = 0 draws nothing: values and gradients pass as they are, infinities and NaN among
them, the same for any seed, and a residual is added once."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("n", [1, 7, 8, 4099])
def test_nothing_is_dropped(n, dtype):
    from gruboros_amd.dropout import dropout

    gen = torch.Generator().manual_seed(n)
    x = torch.randn(n, generator=gen).to(dtype)
    x[0], x[-1] = float("inf"), float("nan")
    x, dy, r = x.to(DEV).requires_grad_(True), torch.randn(n, generator=gen).to(DEV), torch.randn(n, generator=gen).to(DEV)
    for seed in (0, 2 ** 64 - 1, torch.tensor([5], device=DEV)):
        y = dropout(x, 0.0, seed)
        assert torch.equal(y.nan_to_num(7.0), x.nan_to_num(7.0))
        assert torch.equal(torch.autograd.grad(y, x, dy.to(dtype))[0], dy.to(dtype))
        y = dropout(x, 0.0, seed, residual=r)
        assert torch.equal(y.nan_to_num(7.0), (r + x.detach().float()).nan_to_num(7.0))
        assert torch.equal(torch.autograd.grad(y, x, dy)[0], dy.to(dtype))
