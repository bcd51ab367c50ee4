"""The distillation loss's forward and backward in captures of their own."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"


def test_forward_and_backward_in_two_graphs():
    """The backward's graph gives the gradient once however often either is replayed."""
    from gruboros_amd.loss import distillation_loss

    gen = torch.Generator().manual_seed(0)
    z = torch.randn(40, 3001, generator=gen).bfloat16().to(DEV).requires_grad_(True)
    ids, top = torch.randint(0, 3001, (40, 16), generator=gen).to(DEV), torch.randn(40, 16, generator=gen).to(DEV)
    up = torch.tensor(0.5, device=DEV)
    call = lambda: distillation_loss(z, ids, top, temperature=2.0)  # noqa: E731
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        (want,) = torch.autograd.grad(call(), z, up)
    torch.cuda.synchronize()
    ahead, back = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(ahead, stream=side):
        loss = call()
    with torch.cuda.graph(back, stream=side):
        (g,) = torch.autograd.grad(loss, z, up, retain_graph=True)
    for order in ((ahead, back), (back, back), (ahead, back, back)):
        for graph in order:
            graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(g, want)
    (eager,) = torch.autograd.grad(loss, z, up, retain_graph=True)
    back.replay()
    torch.cuda.synchronize()
    assert torch.equal(eager, want) and torch.equal(g, want)
