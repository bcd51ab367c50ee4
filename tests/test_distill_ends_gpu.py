"""Distillation from teachers and of students at the ends of their types, against float64.

Tolerances before any run. The powers' arguments are differences, each rounded once, times a rounded factor: at
|argument| <= 16 off by 3 * 16 * 2^-24 * ln 2 = 2e-6 with exp's 2^-23 beside it; sums of at most 300 terms of one sign
by as much again: 4e-6 of a gradient's terms. bfloat16 half a step, 2^-8, on top. The loss: 1e-5 of its terms' size,
which is its own where one term dwarfs all others.
"""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
f32, bf16 = torch.float32, torch.bfloat16
LOW = {t: torch.finfo(t).min for t in (f32, bf16)}


def _reference(z, ids, top, labels, temperature, alpha):
    """(loss, dz, size of dz's terms) of rows that all count, in float64"""
    z, top = z.double(), top.double()
    p = torch.softmax(top / temperature, -1)
    log_q = torch.log_softmax(z / temperature, -1)
    at = log_q.gather(-1, ids)
    loss = alpha * temperature ** 2 * torch.where(p > 0, p * (p.log() - at), 0.0).sum(-1).mean()
    w = alpha * temperature / len(z)
    q, pr = log_q.exp(), torch.zeros_like(z).scatter_add_(-1, ids, p)
    dz, size = w * (q - pr), w * (q + pr)
    if labels is not None:
        log_q = torch.log_softmax(z, -1)
        loss = loss - (1 - alpha) * log_q.gather(-1, labels[:, None]).mean()
        w = (1 - alpha) / len(z)
        one = torch.nn.functional.one_hot(labels, z.shape[-1])
        dz, size = dz + w * (log_q.exp() - one), size + w * (log_q.exp() + one)
    return float(loss), dz, size


def _check(z, ids, top, labels, temperature, alpha):
    from gruboros_amd.loss import distillation_loss

    zg = z.to(DEV).requires_grad_(True)
    loss = distillation_loss(zg, ids.to(DEV), top.to(DEV), None if labels is None else labels.to(DEV), temperature, alpha)
    want, dz, size = _reference(z, ids, top, labels, temperature, alpha)
    assert abs(float(loss.detach()) - want) <= 1e-5 * (abs(want) + max(temperature ** 2, 1.0)), (float(loss.detach()), want)
    (g,) = torch.autograd.grad(loss, zg)
    err = (g.double().cpu() - dz).abs()
    lim = 4e-6 * size + (2.0 ** -8 if z.dtype == bf16 else 0.0) * dz.abs() + 1e-37
    assert bool((err <= lim).all()), float((err / lim).max())


def _operands(N, V, K, dtype):
    gen = torch.Generator().manual_seed(V + K)
    z = torch.randn(N, V, generator=gen).to(dtype)
    ids = torch.stack([torch.randperm(V, generator=gen)[:K] for _ in range(N)])
    return z, ids, torch.randn(N, K, generator=gen), torch.randint(0, V, (N,), generator=gen)


TYPES = pytest.mark.parametrize("dtype", [f32, bf16], ids=["f32", "bf16"])


@TYPES
@pytest.mark.parametrize("K", [1, 9, 70])
@pytest.mark.parametrize("temperature", [0.25, 1.0, 2.0])
def test_teachers_at_the_ends_of_their_type(temperature, K, dtype):
    """All entries the lowest value (a masked teacher): they share alike; some of them lowest; the largest beside it."""
    z, ids, top, labels = _operands(6, 300, K, dtype)
    for t in (f32, bf16):
        end = top.clone()
        end[0] = end[1] = LOW[t]
        end[1, 0] = 0.0
        end[2, ::2] = LOW[t]
        end[3] = -LOW[t]
        end[4] = LOW[t]
        end[4, -1] = -LOW[t]
        end = end.to(t)
        _check(z, ids, end, labels, temperature, 0.5)
        _check(z, ids, end, None, temperature, 1.0)


@pytest.mark.parametrize("temperature", [1e-3, 0.05, 30.0])
def test_teachers_far_from_zero(temperature):
    """Entries that differ by about a temperature, at a hundred: the difference is what counts."""
    z, ids, top, labels = _operands(6, 300, 20, f32)
    top = 100.0 + temperature * top
    z = (-50.0 + temperature * z).clone()
    _check(z, ids, top, None, temperature, 1.0)
    _check(z, ids, top, labels, temperature, 0.9)


@TYPES
@pytest.mark.parametrize("V,K", [(7, 3), (300, 9), (300, 70), (2500, 20)])
@pytest.mark.parametrize("temperature", [0.5, 1.0, 1.25, 2.0])
def test_students_masked_with_the_lowest_value(temperature, V, K, dtype):
    """A listed or labelled token that the student masks costs its logit's size, which a float holds."""
    z, ids, top, labels = _operands(8, V, K, dtype)
    z[0, ids[0, 0]] = LOW[dtype]
    z[1, labels[1]] = LOW[dtype]
    _check(z, ids, top, None, temperature, 1.0)  # (means over eight rows, which a float holds at these temperatures)
    _check(z, ids, top, labels, temperature, 0.5)
    z[2, ids[2]] = LOW[dtype]
    _check(z, ids, top, labels, temperature, 0.5)
