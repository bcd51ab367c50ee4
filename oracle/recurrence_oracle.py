"""The gated linear recurrence from its definition, token by token (gruboros_amd.recurrence); autograd gives its gradients."""
import torch


def gated_recurrence(x, input_gate, decay_gate, decay, initial_state=None, reset=None, c=8.0):
    """(h [B, T, D], last state [B, D])"""
    rate = torch.nn.functional.softplus(decay, threshold=1e9)
    h = x.new_zeros(x.shape[0], x.shape[2]) if initial_state is None else initial_state
    out = []
    for t in range(x.shape[1]):
        log_a = -c * rate * torch.sigmoid(decay_gate[:, t])
        u = torch.sigmoid(input_gate[:, t]) * x[:, t]
        new = log_a.exp() * h + (-torch.expm1(2.0 * log_a)).sqrt() * u
        h = new if reset is None else torch.where(reset[:, t, None] != 0, u, new)
        out.append(h)
    return (torch.stack(out, 1) if out else x.new_zeros(x.shape)), h
