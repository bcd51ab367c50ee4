"""The gated delta rule token by token, in the inputs' precision (float64 in the tests), on plain
torch operations that autograd differentiates:
    S_t = exp(g_t) S_{t-1} + beta_t k_t (v_t - exp(g_t) S_{t-1}^T k_t)^T,  o_t = scale S_t^T q_t
"""
import torch


def gated_delta_rule(q, k, v, g, beta, state=None, scale=None):
    """q, k [B, T, Hk, K], v [B, T, H, V], g, beta [B, T, H], state [B, H, K, V] or None: (o, last state)."""
    B, T, Hk, K = q.shape
    H, V = v.shape[2:]
    scale = K ** -0.5 if scale is None else scale
    q, k = (x.repeat_interleave(H // Hk, 2) for x in (q, k))
    S = torch.zeros(B, H, K, V, dtype=q.dtype) if state is None else state
    out = []
    for t in range(T):
        S = g[:, t].exp()[..., None, None] * S
        err = v[:, t] - (k[:, t].unsqueeze(-1) * S).sum(-2)
        S = S + (beta[:, t].unsqueeze(-1) * k[:, t]).unsqueeze(-1) * err.unsqueeze(-2)
        out.append(scale * (q[:, t].unsqueeze(-1) * S).sum(-2))
    return torch.stack(out, 1), S
