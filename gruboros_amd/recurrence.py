"""The gated linear recurrence on mg_recurrence_fwd / mg_recurrence_bwd / mg_recurrence_step: a
recurrence like the minGRU's (gruboros_amd.scan) with gates that are not tied to one another. No
counterpart in the reference.

Per batch row and channel, with r = sigmoid(decay_gate_t) and i = sigmoid(input_gate_t),

    a_t = exp(-c softplus(decay) r)
    h_t = a_t h_{t-1} + sqrt(1 - a_t^2) i x_t

``gated_recurrence`` runs whole sequences (training, prompts) with gradients;
``gated_recurrence_step`` one token of generation on a state that it updates in place. Both take
float32 or bfloat16 and keep the state in fp32.
"""
import torch
from torch.autograd import forward_ad

from ._lib import dtype_code, native, no_values, require_cuda, stream_of


def _check(x, input_gate, decay_gate, decay, state, name, dims):
    require_cuda(x, input_gate, decay_gate, decay, state)
    dtype_code(x.dtype)
    if x.dim() != dims:
        raise ValueError(f"x must be [{'B, T, D' if dims == 3 else 'B, D'}], got {tuple(x.shape)}")
    for t, n in ((input_gate, "input_gate"), (decay_gate, "decay_gate")):
        if t.shape != x.shape or t.dtype != x.dtype:
            raise ValueError(f"{n} must be {x.dtype} {tuple(x.shape)} like x, got {t.dtype} {tuple(t.shape)}")
    if not decay.is_floating_point() or decay.shape != x.shape[-1:]:
        raise ValueError(f"decay must be a floating [{x.shape[-1]}] vector, got {decay.dtype} {tuple(decay.shape)}")
    if state is not None and (state.dtype != torch.float32 or state.shape != (x.shape[0], x.shape[-1])):
        raise ValueError(f"{name} must be float32 [{x.shape[0]}, {x.shape[-1]}], got {state.dtype} {tuple(state.shape)}")
    for t in (input_gate, decay_gate, decay, state):
        if t is not None and t.device != x.device:
            raise ValueError(f"operands on {x.device} and {t.device}")


def _rate(c):
    c = float(c)
    if not 0.0 <= c < 1e30:
        raise ValueError(f"c must be in [0, 1e30), got {c}")
    return c


def gated_recurrence(x, input_gate, decay_gate, decay, initial_state=None, reset=None, c=8.0, return_state=False):
    """The gated linear recurrence over sequences.

    x, input_gate, decay_gate [B, T, D] (the gates before their sigmoids), all float32 or all
    bfloat16, with any strides; decay [D], of any floating dtype; initial_state float32 [B, D] or
    None (zeros). reset: bool or uint8 [B, T] or None, nonzero at the first token of each of the
    sequences that are packed into a row: the state before it is forgotten (initial_state too, at
    token 0), whatever it holds, and no gradient crosses it.

    Returns h [B, T, D] in x's dtype, or (h, last state float32 [B, D]) with return_state. Gradients
    reach all tensors but reset, once and in reverse mode. Where they are recorded, the state of
    every eighth token is kept in fp32 for the backward, half a byte per value; a decay gate that is
    shut (its sigmoid is 0 in float32) has no gradient. A value that is not finite
    spoils what follows it in its row and channel, up to the next reset."""
    _check(x, input_gate, decay_gate, decay, initial_state, "initial_state", 3)
    c = _rate(c)
    if reset is not None:
        require_cuda(reset)
        if reset.dtype not in (torch.bool, torch.uint8) or reset.shape != x.shape[:2] or reset.device != x.device:
            raise ValueError(f"reset must be bool or uint8 {tuple(x.shape[:2])} on {x.device}, got {reset.dtype} "
                             f"{tuple(reset.shape)} on {reset.device}")
        reset = reset.contiguous()
    decay = decay.float().contiguous()
    if x.numel() == 0:
        h = no_values(x.new_zeros(x.shape), x, input_gate, decay_gate, decay, initial_state)
        if not return_state:
            return h
        if initial_state is not None:
            return h, initial_state.clone()
        return h, no_values(torch.zeros(x.shape[0], x.shape[2], device=x.device), x, input_gate, decay_gate, decay)
    h0 = None if initial_state is None else initial_state.contiguous()
    h, state = native().recurrence(x, input_gate, decay_gate, decay, h0, reset, c, return_state, stream_of(x))
    return (h, state) if return_state else h


def gated_recurrence_step(x, input_gate, decay_gate, decay, state, c=8.0):
    """One token of the gated linear recurrence, for generation: x, input_gate, decay_gate [B, D] and
    decay [D] as in gated_recurrence, state float32 [B, D], contiguous, which is updated in place.
    Returns h [B, D] in x's dtype. No gradients are recorded: operands that require them are refused
    where they would be."""
    if x.is_cuda and forward_ad._current_level < 0 and 0.0 <= c < 1e30:  # (one call for the operands that generation has)
        h = native().recurrence_step(x, input_gate, decay_gate, decay, state, c, stream_of(x))
        if h is not None:
            return h
    _check(x, input_gate, decay_gate, decay, state, "state", 2)
    c = _rate(c)
    tensors = (x, input_gate, decay_gate, decay, state)
    if torch.is_grad_enabled() and any(t.requires_grad for t in tensors):
        raise ValueError("gated_recurrence_step records no gradients: call it under torch.no_grad(), or use gated_recurrence")
    if forward_ad._current_level >= 0 and any(forward_ad.unpack_dual(t).tangent is not None for t in tensors):
        raise NotImplementedError("the gated linear recurrence has no forward-mode derivative")
    if not state.is_contiguous():
        raise ValueError("state must be contiguous: it is updated in place")
    if x.numel() == 0:
        return torch.empty_like(x)
    x, input_gate, decay_gate = (t.contiguous() for t in (x, input_gate, decay_gate))
    return native().recurrence_step(x, input_gate, decay_gate, decay.float().contiguous(), state, c, stream_of(x))
