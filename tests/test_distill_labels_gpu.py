"""Labels of every integer type that the distillation loss names."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("dtype", [torch.int64, torch.int32, torch.int16, torch.int8, torch.uint8], ids=lambda t: str(t)[6:])
def test_types_of_labels(dtype):
    from gruboros_amd.loss import distillation_loss

    gen = torch.Generator().manual_seed(1)
    z = torch.randn(9, 100, generator=gen).to(DEV)
    ids, top = torch.randint(0, 100, (9, 4), generator=gen).to(DEV), torch.randn(9, 4, generator=gen).to(DEV)
    labels = torch.randint(0, 100, (9,), generator=gen).to(DEV)
    want = distillation_loss(z, ids, top, labels, 2.0, 0.5)
    assert torch.equal(distillation_loss(z, ids, top, labels.to(dtype), 2.0, 0.5), want)
