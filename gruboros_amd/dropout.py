"""Dropout with a counter-based generator (mg_dropout): which values are dropped follows from a
seed, an offset and each value's index (Philox4x32-10), so no mask is stored and the backward
makes the same choice again. Unlike nn.Dropout (reference mingru/minLM.py:72) it draws from no
generator state: a step that is run again, on whatever stream, drops the same values.
"""
import torch

from ._lib import dtype_code, native, no_values, require_cuda, stream_of


def check_drop(p, seed, offset, device):
    """(p, seed as a number, seed as a device tensor or None, offset), checked."""
    p = float(p)
    if not 0.0 <= p < 1.0:
        raise ValueError(f"dropout probability must be in [0, 1), got {p}")
    offset = int(offset)
    if not 0 <= offset < 1 << 64:
        raise ValueError(f"offset must be in [0, 2^64), got {offset}")
    if isinstance(seed, torch.Tensor):
        if seed.dtype != torch.int64 or seed.numel() != 1 or seed.device != device:
            raise ValueError(f"a seed tensor holds one int64 on {device}, got {seed.dtype} {tuple(seed.shape)} on {seed.device}")
        return p, 0, seed, offset
    if seed is None:
        raise ValueError("dropout needs a seed")
    seed = int(seed)
    if not 0 <= seed < 1 << 64:
        raise ValueError(f"seed must be in [0, 2^64), got {seed}")
    return p, seed, None, offset


def _dense(t):
    t = t.contiguous()
    return t.clone() if t.data_ptr() % 16 else t


def dropout(x, p, seed, offset=0, residual=None):
    """x with each value dropped (0) with probability p and the others divided by 1 - p; with
    `residual` (x's shape; float32, or x's dtype) the sum of it and that, in its dtype.

    x: float32 or bfloat16. seed: an integer in [0, 2^64), or one int64 on x's device that the
    kernels read (a replayed graph then sees its current value); offset: an integer that tells the
    calls of one step apart (a layer's number). Value e (row-major) takes word e % 4 of
    Philox4x32-10 at counter (e // 4, offset) under the key seed and is dropped where it is below
    floor(p 2^32). Gradients reach x and residual."""
    require_cuda(x, residual)
    dtype_code(x.dtype)
    p, seed, seed_t, offset = check_drop(p, seed, offset, x.device)
    if residual is not None and (residual.shape != x.shape or residual.dtype not in (torch.float32, x.dtype)
                                 or residual.device != x.device):
        raise ValueError(f"residual {residual.dtype} {tuple(residual.shape)} must match x {tuple(x.shape)}, in float32 or {x.dtype}")
    if x.numel() == 0:
        return x.clone() if residual is None else no_values(residual.clone(), x)
    return native().dropout_add(_dense(x), None if residual is None else _dense(residual), p, seed, seed_t, offset, stream_of(x))
