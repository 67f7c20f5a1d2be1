"""The head's softmax cross entropy from hidden rows and the head's weight, with its
gradient, without the logits tensor (csrc/linear_loss.hip): what scoring and
training need of RMSNorm(x) @ embed^T (model.py:343-348).

Forward leaves each row's log-sum-exp; backward computes the logits again in pieces
of the vocabulary.  The sums are fp32 (over rows: 64 bits, in a fixed order, so a
result does not depend on timing).
"""

import torch

from . import _lib

_REDUCTIONS = ("none", "sum", "mean")


def _forward(hidden, weight, targets, ignore_index, reduction):
    """(nll (T,), lse (T,), loss (), count ()) fp32; loss and count None with "none"."""
    T, (V, H) = hidden.shape[0], weight.shape
    dev, f32 = hidden.device, torch.float32
    nll, lse = torch.empty(T, dtype=f32, device=dev), torch.empty(T, dtype=f32, device=dev)
    loss = count = None
    if reduction:
        loss, count = torch.empty((), dtype=f32, device=dev), torch.empty((), dtype=f32, device=dev)
    if T == 0:
        if reduction:
            loss.fill_(0.0 if reduction == 1 else float("nan"))
            count.zero_()
        return nll, lse, loss, count
    hidden, weight = _lib.rows16(hidden), _lib.rows16(weight)
    with _lib.on_device(hidden):
        n = _lib.workspace_bytes("evo2_linear_loss_workspace_bytes", T, V, H, 0)
        ws = torch.empty(n, dtype=torch.uint8, device=dev)
        _lib.call("evo2_linear_loss", hidden.data_ptr(), hidden.stride(0), weight.data_ptr(),
                  weight.stride(0), targets.data_ptr(), ignore_index, reduction, nll.data_ptr(),
                  lse.data_ptr(), _lib.ptr(loss), _lib.ptr(count), ws.data_ptr(), n, T, V, H,
                  _lib.stream_of(hidden))
    return nll, lse, loss, count


def _backward(ctx, grad):
    hidden, weight, targets, lse, count = ctx.saved_tensors
    T, (V, H) = hidden.shape[0], weight.shape
    need = ctx.needs_input_grad
    dh = hidden.new_empty((T, H)) if need[0] else None
    dw = (weight.new_empty if T else weight.new_zeros)((V, H)) if need[1] else None
    if T:
        hidden, weight = _lib.rows16(hidden), _lib.rows16(weight)
        grad = grad.to(torch.float32)
        with _lib.on_device(hidden):
            n = _lib.workspace_bytes("evo2_linear_loss_workspace_bytes", T, V, H, 1)
            ws = torch.empty(n, dtype=torch.uint8, device=hidden.device)
            _lib.call("evo2_linear_loss_backward", hidden.data_ptr(), hidden.stride(0),
                      weight.data_ptr(), weight.stride(0), targets.data_ptr(), ctx.ignore_index,
                      lse.data_ptr(), grad.data_ptr(), grad.stride(0) if grad.dim() else 0,
                      _lib.ptr(count), _lib.ptr(dh), _lib.ptr(dw), ws.data_ptr(), n, T, V, H,
                      _lib.stream_of(hidden))
    return dh, dw, None, None, None


class _LinearCrossEntropy(torch.autograd.Function):
    @staticmethod
    def forward(ctx, hidden, weight, targets, ignore_index, reduction):
        nll, lse, loss, count = _forward(hidden, weight, targets, ignore_index, reduction)
        ctx.save_for_backward(hidden, weight, targets, lse, count if reduction == 2 else None)
        ctx.ignore_index = ignore_index
        return loss if reduction else nll

    backward = _lib.once(_backward)


def linear_cross_entropy(hidden, weight, targets, ignore_index=-100, reduction="mean"):
    """Cross entropy of the logits hidden @ weight^T against `targets`, differentiable
    in hidden and weight (once).

    hidden (..., H) and weight (V, H) bf16 on one device, H a multiple of 8, V < 2^22; targets
    (...) of an integer type.  Rows whose target is `ignore_index` have loss 0 and no
    gradient (but their infinite or NaN hidden values reach the weight's, times 0); a target
    outside [0, V) otherwise makes its row's loss and gradient NaN (nothing is read
    through it).  reduction: "none" (fp32 losses of targets' shape:
    the negative log-likelihoods), "sum" or "mean" over the rows that are not ignored
    (fp32 scalar; the mean of no rows is NaN).  The logits are fp32 sums of the bf16
    products and never rounded; their gradient (the softmax less one at the target; of
    "none" times the row's upstream gradient) enters the products for hidden and weight as
    bf16, which have fp32 sums."""
    _lib.require_device(hidden, weight, targets)
    if reduction not in _REDUCTIONS:
        raise ValueError(f"reduction must be one of {_REDUCTIONS}, got {reduction!r}")
    if hidden.dtype != torch.bfloat16 or weight.dtype != torch.bfloat16:
        raise ValueError(f"linear_cross_entropy takes bf16 hidden and weight, got {hidden.dtype}, "
                         f"{weight.dtype}")
    if (weight.dim() != 2 or hidden.dim() < 1 or hidden.shape[-1] != weight.shape[1]
            or targets.shape != hidden.shape[:-1]):
        raise ValueError(f"linear_cross_entropy: shapes hidden {tuple(hidden.shape)}, weight "
                         f"{tuple(weight.shape)}, targets {tuple(targets.shape)} do not match")
    if weight.shape[0] == 0 or weight.shape[1] == 0 or weight.shape[1] % 8:
        raise ValueError(f"linear_cross_entropy takes a weight of at least one row and rows of a "
                         f"multiple of 8, got {tuple(weight.shape)}")
    if targets.is_floating_point() or targets.is_complex() or targets.dtype == torch.bool:
        raise ValueError(f"targets must be integers, got {targets.dtype}")
    if not _lib.same_device(hidden, weight, targets):
        raise ValueError(f"linear_cross_entropy: operands on {hidden.device}, {weight.device}, "
                         f"{targets.device}")
    shape = targets.shape
    h = hidden if hidden.dim() == 2 else hidden.reshape(-1, hidden.shape[-1])
    t = targets.reshape(-1).to(torch.int64)
    if t.stride(0) != 1:  # (an expanded target)
        t = t.contiguous()
    red = _REDUCTIONS.index(reduction)
    if _lib.recorded(h, weight):
        out = _LinearCrossEntropy.apply(h, weight, t, int(ignore_index), red)
    else:
        nll, _, loss, _ = _forward(h, weight, t, int(ignore_index), red)
        out = loss if red else nll
    return out if red else out.view(shape)


__all__ = ["linear_cross_entropy"]
