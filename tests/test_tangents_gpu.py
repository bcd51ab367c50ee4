"""Forward-mode differentiation of the gated delta rule, layer norm and dropout: kernels carry no
tangents, so a call on dual tensors is refused, with gradients on and off, instead of returning a
result without its tangent. Plain tensors inside a dual level are no business of it."""
import pytest
import torch
import torch.autograd.forward_ad as fwd

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _calls():
    from gruboros_amd.delta import gated_delta_rule, gated_delta_step
    from gruboros_amd.dropout import dropout
    from gruboros_amd.norm import add_layer_norm, layer_norm

    gen = torch.Generator().manual_seed(0)

    def normal(*s):
        return torch.randn(*s, generator=gen).to(DEV)

    seq = {"q": normal(1, 5, 1, 8), "k": normal(1, 5, 1, 8), "v": normal(1, 5, 2, 8), "g": -normal(1, 5, 2).abs(),
           "beta": normal(1, 5, 2), "initial_state": normal(1, 2, 8, 8)}
    tok = {n: t[:, 0].contiguous() for n, t in seq.items() if n != "initial_state"}
    norm = {"x": normal(3, 16), "w": normal(16), "b": normal(16)}
    return {
        "rule": (lambda **x: gated_delta_rule(**x, return_state=True), seq),
        "step": (lambda **x: gated_delta_step(**x), {**tok, "state": normal(1, 2, 8, 8)}),
        "layer norm": (lambda **x: layer_norm(**x), norm),
        "add layer norm": (lambda **x: add_layer_norm(**x, dropout_p=0.5, seed=1), {**norm, "delta": normal(3, 16)}),
        "dropout": (lambda **x: dropout(**x, p=0.5, seed=1), {"x": normal(3, 16), "residual": normal(3, 16)}),
    }


@pytest.mark.parametrize("grad", [True, False], ids=["grad", "no grad"])
@pytest.mark.parametrize("name", ["rule", "step", "layer norm", "add layer norm", "dropout"])
def test_dual_tensors_are_refused(name, grad):
    call, operands = _calls()[name]
    with torch.set_grad_enabled(grad), fwd.dual_level():
        for n, t in operands.items():
            before = operands["state"].clone() if "state" in operands else None
            with pytest.raises((RuntimeError, NotImplementedError)):
                call(**{**operands, n: fwd.make_dual(t, torch.ones_like(t))})
            assert before is None or torch.equal(operands["state"], before)
        call(**operands)


def test_a_step_of_values_that_are_not_contiguous_is_refused_too():
    call, operands = _calls()["step"]
    wide = operands["v"].repeat(1, 1, 2)[..., :8]
    with torch.no_grad(), fwd.dual_level(), pytest.raises((RuntimeError, NotImplementedError)):
        call(**{**operands, "v": fwd.make_dual(wide, torch.ones_like(wide))})
