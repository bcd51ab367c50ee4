"""The gated delta rule on mg_delta_fwd / mg_delta_bwd / mg_delta_step: a recurrence like the
minGRU's (gruboros_amd.scan) whose state is a matrix. No counterpart in the reference.

Per batch row and head, with a state S [K, V],

    S_t = exp(g_t) S_{t-1} + beta_t k_t (v_t - exp(g_t) S_{t-1}^T k_t)^T
    o_t = scale S_t^T q_t

``gated_delta_rule`` runs whole sequences (training, prompts) in chunks of 64 tokens, with
gradients; ``gated_delta_step`` one token of generation on a state that it updates in place.
Both take float32 or bfloat16 and keep the state in fp32.
"""
import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from ._lib import dtype_code, native, no_values, require_cuda, stream_of


def _operand(t, heads_dim=True):
    """t as the kernels read it: d contiguous, rows (q, k, v, gradients) at multiples of 16 bytes."""
    e = t.element_size()
    if heads_dim:
        if t.stride(-1) != 1 or t.data_ptr() % 16 or any(n > 1 and s * e % 16 for n, s in zip(t.shape[:-1], t.stride())):
            t = t.contiguous()
    if t.shape[1] > 1 and t.stride(1) * e * 64 >= 1 << 31:
        t = t.contiguous()
    return t.clone() if heads_dim and t.data_ptr() % 16 else t


class GatedDeltaRule(torch.autograd.Function):
    """(o, last state or None); see gated_delta_rule."""

    @staticmethod
    def forward(ctx, q, k, v, g, beta, h0, scale, want_state):
        ctx.set_materialize_grads(False)
        o, state, kept = native().delta_fwd(q, k, v, g, beta, h0, scale, want_state, True, stream_of(q))
        ctx.save_for_backward(q, k, v, g, beta, kept)
        ctx.scale = scale
        return o, state

    @staticmethod
    @once_differentiable
    def backward(ctx, do, dstate):
        if do is None and dstate is None:
            return (None,) * 8
        q, k, v, g, beta, kept = ctx.saved_tensors
        do = torch.zeros_like(v, memory_format=torch.contiguous_format) if do is None else _operand(do.to(v.dtype))
        if dstate is not None:
            dstate = dstate.float().contiguous()
        grads = native().delta_bwd(q, k, v, g, beta, ctx.scale, kept, do, dstate, ctx.needs_input_grad[5], stream_of(q))
        return (*(x if need else None for x, need in zip(grads, ctx.needs_input_grad)), None, None)


def _check(q, k, v, g, beta, state, name, lead):
    """Shapes, types and devices; lead: the dimensions before the heads. Tangents, which the kernels do
    not carry, are refused: an operand that has one need not require gradients."""
    require_cuda(q, k, v, g, beta, state)
    dtype_code(q.dtype)
    if q.dim() != lead + 2 or k.shape != q.shape:
        raise ValueError(f"q {tuple(q.shape)} and k {tuple(k.shape)} must both be [{'B, T' if lead == 2 else 'B'}, Hk, K]")
    if v.dim() != lead + 2 or v.shape[:lead] != q.shape[:lead]:
        raise ValueError(f"v {tuple(v.shape)} must be {list(q.shape[:lead])} + [H, V]")
    H, Hk, K, V = v.shape[-2], q.shape[-2], q.shape[-1], v.shape[-1]
    if Hk < 1 or H < 1 or H % Hk:
        raise ValueError(f"the {H} value heads must be a multiple of the {Hk} query/key heads")
    if K % 8 or not 8 <= K <= 128 or V % 8 or not 8 <= V <= 256:
        raise ValueError(f"head sizes K={K}, V={V}: multiples of 8, K <= 128 and V <= 256")
    for t, n in ((g, "g"), (beta, "beta")):
        if t.shape != v.shape[:-1]:
            raise ValueError(f"{n} {tuple(t.shape)} must be {list(v.shape[:-1])}")
    for t, n in ((k, "k"), (v, "v"), (g, "g"), (beta, "beta")):
        if t.dtype != q.dtype:
            raise ValueError(f"{n} is {t.dtype}, q is {q.dtype}: they must share a dtype")
    for t in (k, v, g, beta, state):
        if t is not None and t.device != q.device:
            raise ValueError(f"operands on {q.device} and {t.device}")
    if state is not None and (state.shape != (v.shape[0], H, K, V) or state.dtype != torch.float32):
        raise ValueError(f"{name} must be float32 [{v.shape[0]}, {H}, {K}, {V}], got {state.dtype} {tuple(state.shape)}")
    if forward_ad._current_level >= 0 and any(t is not None and forward_ad.unpack_dual(t).tangent is not None
                                              for t in (q, k, v, g, beta, state)):
        raise NotImplementedError("the gated delta rule has no forward-mode derivative")


def gated_delta_rule(q, k, v, g, beta, initial_state=None, scale=None, return_state=False):
    """The gated delta rule over sequences.

    q, k [B, T, Hk, K], v [B, T, H, V], g (log decay) and beta (write strength) [B, T, H], all
    float32 or all bfloat16, with any strides; H a multiple of Hk: value head h reads q and k of
    head h // (H // Hk). K and V are multiples of 8, K <= 128, V <= 256. initial_state: float32
    [B, H, K, V] or None (zeros). scale: K ** -0.5 by default. g = -inf forgets the state.

    Returns o [B, T, H, V] in the inputs' dtype, or (o, last state float32 [B, H, K, V]) with
    return_state. Gradients reach all six tensors, once and in reverse mode (no double backward, and
    dual tensors are refused). Where gradients are recorded, each 64 tokens of a head keep their
    state, updates and operands for the backward: 4 K V + 256 V + 134700 bytes for K > 64, 101900 in
    place of the last for K <= 64 (float32: 6 K V + 384 V + 271900 or 173600), with K rounded up to
    64 or 128 and V to a multiple of 32. Without, a call takes 81408 or 56832 bytes (float32: 185856 or
    112128) for as long as it runs.

    The 64 tokens of a chunk are solved as a triangular system, whose condition grows with beta |k|^2
    where keys are alike: all keys the same, float32 is off by 1e-6 at 1, by 2e-4 at 2.

    A value that is not finite spoils the 64 tokens of its chunk, earlier ones included: padding
    behind a sequence must be finite."""
    _check(q, k, v, g, beta, initial_state, "initial_state", 2)
    scale = q.shape[-1] ** -0.5 if scale is None else float(scale)
    if q.shape[0] == 0 or q.shape[1] == 0:  # no token: nothing is written
        o = no_values(v.new_zeros(v.shape), q, k, v, g, beta, initial_state)
        if not return_state:
            return o
        size = (v.shape[0], v.shape[2], q.shape[3], v.shape[3])
        state = torch.zeros(size, device=v.device) if initial_state is None else initial_state.clone()
        return o, (state if q.shape[0] else no_values(state, q, k, v, g, beta))
    q, k, v = _operand(q), _operand(k), _operand(v)
    g, beta = _operand(g, False), _operand(beta, False)
    h0 = None if initial_state is None else initial_state.contiguous()
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (q, k, v, g, beta, h0)):
        o, state = GatedDeltaRule.apply(q, k, v, g, beta, h0, scale, return_state)
    else:
        o, state, _ = native().delta_fwd(q, k, v, g, beta, h0, scale, return_state, False, stream_of(q))
    return (o, state) if return_state else o


def gated_delta_step(q, k, v, g, beta, state, scale=None):
    """One token of the gated delta rule, for generation: q, k [B, Hk, K], v [B, H, V], g and beta
    [B, H] as in gated_delta_rule, state float32 [B, H, K, V], contiguous, which is updated in
    place. Returns o [B, H, V]. No gradients are recorded: operands that require them are refused
    where they would be."""
    if q.is_cuda and forward_ad._current_level < 0:  # (one call for the operands that generation has)
        o = native().delta_step_plain(q, k, v, g, beta, state, scale, stream_of(q))
        if o is not None:
            return o
    _check(q, k, v, g, beta, state, "state", 1)
    if torch.is_grad_enabled() and any(t.requires_grad for t in (q, k, v, g, beta, state)):
        raise ValueError("gated_delta_step records no gradients: call it under torch.no_grad(), or use gated_delta_rule")
    if not state.is_contiguous() or state.data_ptr() % 16:
        raise ValueError("state must be contiguous and 16-byte aligned: it is updated in place")
    if v.shape[0] == 0:
        return torch.empty_like(v)
    q, k, v, g, beta = (t.contiguous() for t in (q, k, v, g, beta))
    if v.data_ptr() % 16:
        v = v.clone()
    o = native().delta_step(q, k, v, g, beta, state, q.shape[-1] ** -0.5 if scale is None else float(scale), stream_of(q))
    if not state.is_inference():
        torch.autograd.graph.increment_version(state)
    return o
