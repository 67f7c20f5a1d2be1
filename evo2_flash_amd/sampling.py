"""The next token from the logits (csrc/sample.hip): temperature, top-k, top-p and min-p, and
the draw from given uniform numbers, behind the decoder's head (model.py:343-348).
"""

from operator import index

import torch

from . import _lib


_TYPES = (torch.bfloat16, torch.float32)


def _setting(x, name, B, dev, dtype):
    """(address or None, number) of a setting: a tensor (B,) on device `dev`, or one number
    for all rows; and the tensor, to be kept until the launch."""
    if not isinstance(x, torch.Tensor):
        return None, min(max(index(x), 0), 2 ** 31 - 1) if dtype is torch.int32 else float(x), None
    if x.shape != (B,):
        raise ValueError(f"{name} must be one number or ({B},), got {tuple(x.shape)}")
    if x.get_device() != dev:
        raise ValueError(f"{name} is on {x.device}, the logits on cuda:{dev}")
    if x.dtype != dtype:
        if dtype is torch.int32:
            if x.dtype != torch.int64:
                raise ValueError(f"{name} must be int32 or int64, got {x.dtype}")
            x = x.clamp(0, 2 ** 31 - 1)
        elif not x.is_floating_point():
            raise ValueError(f"{name} must be floating-point numbers, got {x.dtype}")
        x = x.to(dtype)
    if B > 1 and x.stride(0) != 1:
        x = x.contiguous()
    return x.data_ptr(), 0, x


def sample_tokens(logits, uniforms, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """The next token of each row: logits (B, V) bf16 or fp32 (rows of any stride),
    uniforms (B,) fp32 numbers of [0, 1) -> (B,) int64.  temperature, top_k, top_p and min_p
    are one number each or (B,) tensors on the logits' device (the host does not read those);
    they are taken as fp32 and int32.

    The tokens stand in the order of their logits, equal ones the lowest index first.
    top_k > 0 keeps the first top_k; top_p < 1 the shortest front of those whose
    probabilities (softmax(logits / temperature), of what top_k kept) reach top_p, at least
    the first token; min_p > 0 those with at least min_p (at most 1) times the largest
    probability.  The token is the first, in the vocabulary's order, at which the running sum
    of what is kept passes uniforms times its total; numbers outside [0, 1) draw the first or
    the last token kept.  temperature <= 0 (or NaN) and top_k 1 take the first token.  -inf and
    NaN logits are never drawn (a row of nothing else gives -1); beside +inf no finite one
    is.  Weights are summed as whole numbers, so a result does not depend on timing, and tokens
    that are all equal are parted exactly.  A token of less than 2^-50 of the largest weight (V
    over 8192: V 2^-62) may count for nothing; a running sum, and so the border between two
    tokens, is off by at most V 2^-48 of the total.  More than 65535 rows are refused where a
    row has more than 4096 logits."""
    shape, dtype, dev = logits.shape, logits.dtype, logits.get_device()
    same = uniforms.get_device() == dev
    if dev < 0 or not same:
        _lib.require_device(logits, uniforms)
        if not same:
            raise ValueError(f"uniforms are on {uniforms.device}, the logits on {logits.device}")
    if len(shape) != 2 or dtype not in _TYPES:
        raise ValueError(f"sample_tokens takes bf16 or fp32 logits (B, V), got {tuple(shape)} {dtype}")
    B, V = shape
    if not 0 < V <= 1 << 20:
        raise ValueError(f"sample_tokens takes 1 to 2^20 logits a row, got {V}")
    if uniforms.shape != (B,) or uniforms.dtype != torch.float32:
        raise ValueError(f"uniforms must be ({B},) fp32, got {tuple(uniforms.shape)} {uniforms.dtype}")
    t, t1, keep_t = _setting(temperature, "temperature", B, dev, torch.float32)
    k, k1, keep_k = _setting(top_k, "top_k", B, dev, torch.int32)
    p, p1, keep_p = _setting(top_p, "top_p", B, dev, torch.float32)
    m, m1, keep_m = _setting(min_p, "min_p", B, dev, torch.float32)
    out = torch.empty(B, dtype=torch.int64, device=logits.device)
    if B == 0:
        return out
    row, unit = logits.stride()
    if unit != 1 or (row < V and B > 1):
        logits = logits.contiguous()
        row = logits.stride(0)
    if B > 1 and uniforms.stride(0) != 1:
        uniforms = uniforms.contiguous()
    with _lib.on_device(logits):
        bytes = _lib.workspace_bytes("evo2_sample_workspace_bytes", B, V)
        work = torch.empty(bytes, dtype=torch.uint8, device=logits.device) if bytes else None
        _lib.call("evo2_sample", logits.data_ptr(), dtype == torch.float32, row, uniforms.data_ptr(), t, t1,
                  k, k1, p, p1, m, m1, _lib.ptr(work), bytes, out.data_ptr(), B, V, _lib.stream_of(logits))
    return out


__all__ = ["sample_tokens"]
