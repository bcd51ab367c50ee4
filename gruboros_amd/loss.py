"""Loss head: logits projection + mean cross-entropy (reference
mingru/minLM.py:138, :146-149). For bf16 embeddings and V <= 256 classes the
logits product, log-softmax, loss and logits gradient are one kernel
(mg_logits_cross_entropy) and the fp32 logits never reach memory; otherwise
the logits are formed first and mg_cross_entropy_fwd_bwd does the rest in one
pass. distillation_loss (mg_distill) is the loss of a student that learns from
a teacher's top logits, and from labels beside them, for any vocabulary.
"""
import torch

from . import gemm
from ._lib import check, dtype_code, lib, native, no_values, ptr, require_cuda, stream_of
from .linear import _mm_f32, bf16_copy, f32_linear, f32_linear_applies


def _ce(logits2d, labels1d, grad_dtype):
    N, V = logits2d.shape
    L = lib()
    P = L.mg_cross_entropy_partials(N)
    dl = torch.empty(N, V, dtype=grad_dtype, device=logits2d.device)
    part = torch.empty(P, dtype=torch.float32, device=logits2d.device)
    rc = L.mg_cross_entropy_fwd_bwd(dtype_code(logits2d.dtype), ptr(logits2d), ptr(labels1d), dtype_code(grad_dtype),
                                    ptr(dl), ptr(part), None, N, V, 1.0 / N, stream_of(logits2d))
    check(rc, "mg_cross_entropy_fwd_bwd")
    return part.sum() / N, dl


class LogitsCrossEntropy(torch.autograd.Function):
    """mean_n CE(embed_n @ W^T, label_n); embed bf16 [N, D], W fp32 master [V, D]."""

    @staticmethod
    def forward(ctx, embed, w, wb, labels):
        N, D = embed.shape
        V = wb.shape[0]
        if V <= 256 and V % 8 == 0 and D % 8 == 0:
            L = lib()
            dl = torch.empty(N, V, dtype=torch.bfloat16, device=embed.device)
            part = torch.empty(L.mg_logits_cross_entropy_partials(N), dtype=torch.float32, device=embed.device)
            rc = L.mg_logits_cross_entropy(ptr(embed), embed.stride(0), ptr(wb), wb.stride(0), ptr(labels), ptr(dl),
                                           V, ptr(part), None, N, D, V, 1.0 / N, stream_of(embed))
            check(rc, "mg_logits_cross_entropy")
            loss = part.sum() / N
        else:
            logits = _mm_f32(embed, wb.t())               # [N, V] fp32
            loss, dl = _ce(logits, labels, torch.bfloat16)
        ctx.save_for_backward(embed, wb, dl)
        return loss

    @staticmethod
    def backward(ctx, g):
        embed, wb, dl = ctx.saved_tensors
        dl = dl * g  # upstream gradient (1/grad_accum in the reference loop); stays bf16
        de = torch.mm(dl, wb) if ctx.needs_input_grad[0] else None
        dw = gemm.linear_dw(dl, embed) if ctx.needs_input_grad[1] else None
        return de, dw, None, None


class CrossEntropyFromLogits(torch.autograd.Function):
    """mean_n CE(logits_n, label_n) for fp32 logits [N, V] (the fp32 path)."""

    @staticmethod
    def forward(ctx, logits, labels):
        loss, dl = _ce(logits, labels, torch.float32)
        ctx.save_for_backward(dl)
        return loss

    @staticmethod
    def backward(ctx, g):
        (dl,) = ctx.saved_tensors
        return dl * g, None


def logits_cross_entropy(embed, to_logits, labels):
    """Mean cross-entropy of to_logits(embed) against labels (int64), like
    F.cross_entropy(logits.transpose(1, 2), labels) in the reference."""
    require_cuda(embed, labels)
    D = embed.shape[-1]
    e2 = embed.reshape(-1, D)
    lab = labels.reshape(-1).contiguous()
    w = to_logits.weight
    if embed.dtype == torch.bfloat16 and w.dtype == torch.float32:
        return LogitsCrossEntropy.apply(e2.contiguous(), w, bf16_copy(w), lab)
    if f32_linear_applies(e2, w):
        logits = f32_linear(e2, w)  # the fp32 path: the logits product on mg_gemm_f32
    else:
        logits = torch.nn.functional.linear(e2.to(w.dtype), w)  # (parameters cast to another dtype: product in it)
    return CrossEntropyFromLogits.apply(logits.float().contiguous(), lab)


def distillation_loss(logits, top_ids, top_logits, labels=None, temperature=1.0, alpha=1.0):
    """The loss of a student that learns from a teacher's K largest logits per token, and from labels:

        alpha * temperature^2 * mean KL(softmax(top_logits / temperature) || softmax(logits / temperature)[top_ids])
        + (1 - alpha) * mean cross_entropy(logits, labels)

    logits [N, V] or [B, T, V] (float32 or bfloat16; batch and steps may be strided, as in
    logits[:, :-1]), top_ids (int64 or int32) and top_logits (float32 or bfloat16) [..., K] with
    1 <= K <= 512, labels [...] (int64, int32, int16, int8 or uint8) or None where alpha is 1. The
    teacher's distribution is over its K entries alone; one whose id is outside [0, V) or whose logit
    is -inf is none, and an id that is listed twice counts twice. Rows without an entry, and labels
    outside [0, V) such as -100, do not count: each mean is over the rows that do, and 0 where none
    does. What a row that counts for neither holds does not matter.

    Returns the loss, a float32 scalar. The gradient reaches logits, in their dtype, once and in
    reverse mode; it is made in the forward's pass and kept until the backward, which multiplies it
    by the loss's own gradient (in bfloat16 that rounds a second time, unless it is a power of two),
    and which makes it again where it is run a second time over a retained graph, or in another
    captured graph than the forward."""
    require_cuda(logits, top_ids, top_logits, labels)
    dtype_code(logits.dtype)
    dtype_code(top_logits.dtype)
    if logits.dim() not in (2, 3) or not 1 <= logits.shape[-1] <= 1 << 30:
        raise ValueError(f"logits must be [N, V] or [B, T, V] with 1 <= V <= 2^30, got {tuple(logits.shape)}")
    if top_ids.dtype not in (torch.int64, torch.int32):
        raise ValueError(f"top_ids must be int64 or int32, got {top_ids.dtype}")
    if top_ids.shape[:-1] != logits.shape[:-1] or top_ids.dim() != logits.dim() or not 1 <= top_ids.shape[-1] <= 512:
        raise ValueError(f"top_ids must be {list(logits.shape[:-1])} + [K], 1 <= K <= 512, got {tuple(top_ids.shape)}")
    if top_logits.shape != top_ids.shape:
        raise ValueError(f"top_logits {tuple(top_logits.shape)} must match top_ids {tuple(top_ids.shape)}")
    temperature, alpha = float(temperature), float(alpha)
    if not 1e-4 <= temperature <= 1e4:
        raise ValueError(f"temperature must be in [1e-4, 1e4], got {temperature}")
    if not 0.0 <= alpha <= 1.0:
        raise ValueError(f"alpha must be in [0, 1], got {alpha}")
    if labels is None:
        if alpha != 1.0:
            raise ValueError(f"alpha {alpha} gives the labels a share of the loss: labels are needed")
    elif labels.shape != logits.shape[:-1] or labels.dtype not in (torch.int64, torch.int32, torch.int16, torch.int8, torch.uint8):
        raise ValueError(f"labels must be integers {list(logits.shape[:-1])}, got {labels.dtype} {tuple(labels.shape)}")
    for t in (top_ids, top_logits, labels):
        if t is not None and t.device != logits.device:
            raise ValueError(f"operands on {logits.device} and {t.device}")
    if torch.is_grad_enabled() and top_logits.requires_grad:
        raise ValueError("no gradient reaches the teacher: detach top_logits")
    if logits.numel() == 0:
        return no_values(torch.zeros((), device=logits.device), logits)
    if logits.numel() // logits.shape[-1] >= 1 << 31:
        raise ValueError("a call takes fewer than 2^31 rows")
    labels = None if labels is None else labels.long()
    return native().distill(logits, top_ids, top_logits, labels, temperature, alpha, stream_of(logits))
