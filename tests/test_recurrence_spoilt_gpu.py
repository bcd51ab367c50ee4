"""The gated linear recurrence where a state is not finite and forgotten fast: products of decays that
underflow to 0 drop finite values only, a reset drops all. What is spoilt is told token by token."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
f32, bf16 = torch.float32, torch.bfloat16
NAMES = ("x", "input_gate", "decay_gate", "decay", "initial_state")


def _operands(B, T, D, dtype, log_a):
    """Operands whose gates are shut and open about as often; the decay is log_a at an open gate of 30 and more"""
    gen = torch.Generator().manual_seed(T)
    n = lambda *s: torch.randn(*s, generator=gen)  # noqa: E731
    rate = torch.tensor(-log_a / 8.0, dtype=torch.float64)
    return {"x": n(B, T, D).to(dtype), "input_gate": n(B, T, D).to(dtype), "decay_gate": torch.full((B, T, D), 40.0, dtype=dtype),
            "decay": torch.log(torch.expm1(rate)).float().expand(D).clone(), "initial_state": n(B, D)}, n(B, T, D).to(dtype)


def _place(ops):
    return {k: v.to(DEV).requires_grad_(True) for k, v in ops.items()}


LOG_A = pytest.mark.parametrize("log_a", [-11.0, -4.0, -1.0, -0.2])
TYPES = pytest.mark.parametrize("dtype", [f32, bf16], ids=["f32", "bf16"])


@TYPES
@LOG_A
@pytest.mark.parametrize("value", ["nan", "inf", "-inf"])
def test_marks_that_are_all_zero_are_none(value, log_a, dtype):
    """What is not finite at token 10 spoils its row and channel from there to the end, the state too."""
    from gruboros_amd.recurrence import gated_recurrence

    T = 700
    ops, _ = _operands(2, T, 70, dtype, log_a)
    ops["x"][1, 10, 3] = float(value)
    dev = {k: v.to(DEV) for k, v in ops.items()}
    zero = torch.zeros(2, T, dtype=torch.bool, device=DEV)
    for reset in (None, zero):
        h, last = gated_recurrence(**dev, reset=reset, return_state=True)
        bad = ~torch.isfinite(h)
        want = torch.zeros_like(bad)
        want[1, 10:, 3] = True
        assert torch.equal(bad, want)
        assert torch.equal(~torch.isfinite(last), want[:, -1])


@TYPES
@LOG_A
def test_a_state_that_is_nan(log_a, dtype):
    """A state that is carried in is told to the end, or to the first mark, in whichever tile that is."""
    from gruboros_amd.recurrence import gated_recurrence

    T = 900
    ops, _ = _operands(3, T, 5, dtype, log_a)
    clean = {k: v.to(DEV) for k, v in ops.items()}
    reset = torch.zeros(3, T, dtype=torch.bool, device=DEV)
    reset[0, 5], reset[1, 511] = True, True
    h = gated_recurrence(**clean, reset=reset)
    bad = {**clean, "initial_state": torch.full_like(clean["initial_state"], float("nan"))}
    hb, last = gated_recurrence(**bad, reset=reset, return_state=True)
    for b, n in enumerate((5, 511, T)):
        assert bool(torch.isnan(hb[b, :n]).all()) and torch.equal(hb[b, n:], h[b, n:])
    assert torch.equal(torch.isnan(last).all(-1).cpu(), torch.tensor([False, False, True]))


@TYPES
@LOG_A
@pytest.mark.parametrize("bits", [0x7FC00000, 0xFFC00000], ids=["nan", "-nan"])
def test_a_gate_that_is_nan(bits, log_a, dtype):
    """A decay that is NaN, of either sign, is no reset: all is spoilt up to the next one."""
    from gruboros_amd.recurrence import gated_recurrence

    T = 500
    ops, dh = _operands(1, T, 6, dtype, log_a)
    reset = torch.zeros(1, T, dtype=torch.bool, device=DEV)
    reset[0, [100, 300]] = True
    clean = _place(ops)
    nan = torch.tensor([bits - (1 << 32) if bits >> 31 else bits], dtype=torch.int32).view(f32)
    if dtype == bf16:
        nan = torch.tensor([(bits >> 16) - (1 << 16) if bits >> 31 else bits >> 16], dtype=torch.int16).view(bf16)
    ops["decay_gate"][0, 150] = nan
    dev = _place(ops)
    h, hb = gated_recurrence(**clean, reset=reset), gated_recurrence(**dev, reset=reset)
    assert torch.equal(hb[:, :150], h[:, :150]) and torch.equal(hb[:, 300:], h[:, 300:])
    assert bool(torch.isnan(hb[:, 150:300]).all())
    # the state before it reaches no later gradient but through it
    gb = torch.autograd.grad(hb, dev["x"], dh.to(DEV))[0]
    g = torch.autograd.grad(h, clean["x"], dh.to(DEV))[0]
    assert bool(torch.isnan(gb[:, 100:151]).all())
    for part in (slice(0, 100), slice(151, T)):
        assert torch.equal(gb[:, part], g[:, part])


@TYPES
@LOG_A
def test_gradients(log_a, dtype):
    """A gradient that is NaN spoils those of all tokens before it, back to the mark or to the state."""
    from gruboros_amd.recurrence import gated_recurrence

    T = 700
    ops, dh = _operands(2, T, 70, dtype, log_a)
    reset = torch.zeros(2, T, dtype=torch.bool, device=DEV)
    reset[1, 130] = True
    dev = _place(ops)
    leaves = [dev[k] for k in NAMES]
    clean = torch.autograd.grad(gated_recurrence(**dev, reset=reset), leaves, dh.to(DEV))
    dh[:, 600, 3] = float("nan")
    for marks in (None, reset):
        g = torch.autograd.grad(gated_recurrence(**dev, reset=marks), leaves, dh.to(DEV))
        want = torch.zeros(2, T, 70, dtype=torch.bool, device=DEV)
        want[0, :601, 3] = True
        want[1, 0 if marks is None else 130:601, 3] = True
        for i in range(2):
            assert torch.equal(torch.isnan(g[i]), want), NAMES[i]
        # (the token of a mark has no gradient to its decay gate)
        gate = want.clone()
        if marks is not None:
            gate[1, 130] = False
        assert torch.equal(torch.isnan(g[2]), gate)
        assert torch.equal(torch.isnan(g[4][:, 3]).cpu(), torch.tensor([True, marks is None]))
        assert bool(torch.isfinite(g[4][:, 4:]).all())
    for i in range(3):
        assert torch.equal(g[i][~want], clean[i][~want])
