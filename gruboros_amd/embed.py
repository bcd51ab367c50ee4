"""Token embedding with the weight gradient on mg_embedding_bwd.

Reference mingru/minLM.py:92,99: `nn.Embedding(num_tokens, dim)` looked up on
the token ids. The forward is torch's gather (it also refuses ids outside the
table). The backward, dw[v] = sum of the output-gradient rows of the tokens
with id v, runs on three kernels that sum in a fixed order and never copy
anything to the host. torch's embedding backward copies a segment count to the
host, which holds the host at the end of every backward pass while the GPU
drains; the optimizer's host work then ran with the GPU idle (0.12-0.2 ms per
cfg3 step, beside the 0.12 ms of the backward's own kernels).

scaled_embedding (mg_embedding_fwd / mg_embedding_sorted_bwd) is the same for
any vocabulary and table type, with a scale: lookup, scale and cast in one
pass, and a gradient by tokens sorted on the GPU.
"""
import torch
import torch.nn.functional as F

from ._lib import check, dtype_code, lib, native, no_values, ptr, require_cuda, stream_of

MAX_VOCAB = 512  # mg_embedding_bwd's table limit


class EmbeddingFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, ids, weight):
        ids = ids.contiguous()  # (a slice of the batch: one copy, shared by the gather and the backward)
        ctx.save_for_backward(ids)
        ctx.vd = tuple(weight.shape)
        return F.embedding(ids, weight)

    @staticmethod
    def backward(ctx, dy):
        (ids,) = ctx.saved_tensors
        V, D = ctx.vd
        dx = dy.reshape(-1, D)
        if dx.dtype != torch.float32 or dx.stride(1) != 1 or dx.stride(0) % 4 or dx.data_ptr() % 16:
            dx = dx.float().contiguous()
        flat = ids.reshape(-1)
        if not flat.is_contiguous():
            flat = flat.contiguous()
        N = flat.numel()
        dw = torch.empty(V, D, dtype=torch.float32, device=dx.device)
        L = lib()
        ws = torch.empty(L.mg_embedding_bwd_workspace_bytes(N, D, V), dtype=torch.uint8, device=dx.device)
        check(L.mg_embedding_bwd(ptr(flat), ptr(dx), dx.stride(0), N, D, V, ptr(dw), D, ptr(ws), ws.numel(),
                                 stream_of(dx)), "mg_embedding_bwd")
        return None, dw


def embedding(ids: torch.Tensor, weight: torch.Tensor) -> torch.Tensor:
    """F.embedding(ids, weight); the weight gradient of an fp32 table of at most
    MAX_VOCAB rows (the reference's byte vocabulary is 256) goes through
    mg_embedding_bwd, other tables through torch's backward."""
    V, D = weight.shape
    if (torch.is_grad_enabled() and weight.requires_grad and weight.is_cuda and weight.dtype == torch.float32
            and ids.dtype == torch.int64 and 1 <= V <= MAX_VOCAB and D % 4 == 0 and ids.numel() > 0
            and ids.numel() < (1 << 31)):
        return EmbeddingFn.apply(ids, weight)
    return F.embedding(ids, weight)


def scaled_embedding(ids, weight, scale=1.0, out_dtype=None, padding_idx=None):
    """scale * weight[ids] in out_dtype (default weight's), for tables of any size.

    ids: int64 or int32 of any shape; weight [V, D], float32 or bfloat16, V < 2^28, D < 2^30; fewer
    than 2^27 ids. The gradient reaches weight, in its dtype, once and in reverse mode: rows are
    summed in fp32 in the order of the tokens and rounded once, so results repeat bit for bit. An id
    outside the table (torch's lookup stops the process there) gives a row of NaN and no gradient.
    The row of padding_idx, which counts from the end where it is negative, gets no gradient."""
    require_cuda(ids, weight)
    if ids.dtype not in (torch.int64, torch.int32):
        raise ValueError(f"ids must be int64 or int32, got {ids.dtype}")
    if weight.dim() != 2 or not 1 <= weight.shape[0] < 1 << 28 or weight.shape[1] >= 1 << 30:
        raise ValueError(f"weight must be [V, D] with 1 <= V < 2^28 and D < 2^30, got {tuple(weight.shape)}")
    if ids.numel() >= 1 << 27:
        raise ValueError(f"{ids.numel()} ids: a call takes fewer than 2^27")
    if ids.device != weight.device:
        raise ValueError(f"operands on {ids.device} and {weight.device}")
    dtype_code(weight.dtype)
    out_dtype = out_dtype or weight.dtype
    dtype_code(out_dtype)
    V, D = weight.shape
    scale = float(scale)
    padding = -1
    if padding_idx is not None:
        if not -V <= padding_idx < V:
            raise ValueError(f"padding_idx {padding_idx} is outside a table of {V} rows")
        padding = int(padding_idx) % V
    if ids.numel() == 0 or D == 0:
        return no_values(torch.empty(*ids.shape, D, dtype=out_dtype, device=weight.device), weight)
    return native().scaled_embedding(ids, weight, scale, out_dtype == torch.bfloat16, padding, stream_of(weight))
