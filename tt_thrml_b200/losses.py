"""Softmax cross entropy of categories that are read out of a block's units.

    l[t, v] = sum_k x[t, k] w[v, k] + bias[v],   loss[t] = log sum_v exp l[t, v] - l[t, y[t]]

The logits are never held as a whole: the forward pass keeps a running maximum
and sum per row, the backward pass takes the categories in pieces: 256 MiB of
16-bit differences exp(l - z) - [v = y] at a time, or 512 bytes a row where that is
more.  x is a dense
block's units over the chains (or any features), w one row per category.

The kernels launch on the current stream of x's device; nothing synchronises.
A kernel whose wait expires (two seconds) gives up and leaves a code that
check_operator_errors reports.
"""

from __future__ import annotations

from . import _native as nat
from .quantized import _error_addresses, dtype_code, error_word, on_device, require_cuda

_REDUCTIONS = {"none": 0, "mean": 1, "sum": 2}


def _torch():
    import torch

    return torch


def _check(x, weights, targets, bias) -> None:
    torch = _torch()
    require_cuda("x", x)
    dev = x.device
    if dtype_code(x.dtype) not in (nat.DT_BF16, nat.DT_F16) or x.dim() < 1:
        raise ValueError(f"x must hold bfloat16 or float16 rows, got {x.dtype} of shape {tuple(x.shape)}")
    require_cuda("weights", weights, dev)
    if weights.dtype != x.dtype or weights.dim() != 2:
        raise ValueError(f"weights must be a {x.dtype} matrix, got {weights.dtype} of shape {tuple(weights.shape)}")
    V, K = weights.shape
    if x.shape[-1] != K:
        raise ValueError(f"x has rows of {x.shape[-1]}, the weights have {K} columns")
    if not (1 <= V <= nat.XENT_MAX_CATEGORIES and 1 <= K <= nat.XENT_MAX_COLS):
        raise ValueError(f"1 to {nat.XENT_MAX_CATEGORIES} categories of 1 to {nat.XENT_MAX_COLS} columns are supported, "
                         f"got {V} of {K}")
    require_cuda("targets", targets, dev)
    if targets.dtype not in (torch.int64, torch.int32) or targets.shape != x.shape[:-1]:
        raise ValueError(f"targets must be int64 or int32 of shape {tuple(x.shape[:-1])}, got {targets.dtype} of "
                         f"{tuple(targets.shape)}")
    if bias is not None:
        require_cuda("bias", bias, dev)
        if bias.dtype != torch.float32 or bias.shape != (V,):
            raise ValueError(f"bias must be float32 of shape ({V},), got {bias.dtype} of {tuple(bias.shape)}")
    rows = targets.numel()
    if rows > nat.XENT_MAX_ROWS:
        raise ValueError(f"at most {nat.XENT_MAX_ROWS} rows are supported, got {rows}")


def mean_and_gradients(x, weights, targets, bias, ignore_index, one, dw, db):
    """The mean loss of x [rows, K], a float32 scalar on the device, with its gradients written into dw [V, K] (float32 or
    weights' type, dense) and db; nothing of it is recorded for autograd.  one: the float32 number 1 on x's device."""
    _check(x, weights, targets, bias)
    if x.dim() != 2 or not x.shape[0]:
        raise ValueError(f"x must hold rows of units, got shape {tuple(x.shape)}")
    word = _error_addresses.get(x.device.index) or error_word(x.device).data_ptr()
    with on_device(x.device):
        return nat.bound_hostcall().softmax_cross_entropy_gradients(x, weights, bias, targets, int(ignore_index), word, one, dw, db)


def softmax_cross_entropy(x, weights, targets, *, bias=None, reduction="mean", ignore_index=-100):
    """Minus the log likelihood of the target categories under softmax(x weights^T + bias), differentiable in x, weights
    and bias.

    x: bfloat16 or float16 [..., K]; weights: the same type [V, K], any strides
    (rows that are not 16-byte aligned are laid out again in each call); targets:
    int64 or int32 [...]; bias: float32 [V], -inf for categories that cannot occur, whose
    weights must be finite all the same (logits below -2^127 may count as -inf).
    reduction "mean" (over the rows that count), "sum" (float32 scalars) or "none"
    (float32 [...]).  Rows whose target is `ignore_index` do not count: loss 0, no
    gradient (their values must be finite, as 0 times them is added to the weights'
    gradient); a mean over no rows is 0.  A target outside 0 .. V - 1 gives NaN.  A
    row in which no category can occur has loss inf and no gradient.

    Sums and normalisers are float32; the gradients are products of 16-bit
    differences, accumulated in float32 (in float16 the differences are held relative
    to the largest weight of a row under 'none': below 2^-28 of it they lose bits).
    The result is the same every time, whichever gradients are asked for.
    Gradients of gradients and forward-mode derivatives are not available.
    """
    torch = _torch()
    _check(x, weights, targets, bias)
    V, K = weights.shape
    dev = x.device
    if reduction not in _REDUCTIONS:
        raise ValueError(f"reduction must be 'mean', 'sum' or 'none', got {reduction!r}")
    lead = x.shape[:-1]
    rows = targets.numel()
    if rows == 0:  # nothing counts
        zero = x.sum(-1).float() + weights[:0].sum().float() + (0.0 if bias is None else bias[:0].sum())
        return zero if reduction == "none" else zero.sum()
    word = _error_addresses.get(dev.index) or error_word(dev).data_ptr()
    flat = x if x.dim() == 2 else x.reshape(rows, K)
    targets = targets if targets.dim() == 1 else targets.reshape(rows)
    with on_device(dev):
        loss = nat.bound_hostcall().softmax_cross_entropy(flat, weights, bias, targets, _REDUCTIONS[reduction], int(ignore_index),
                                                          word)
    return loss.reshape(lead) if reduction == "none" and len(lead) != 1 else loss


__all__ = ["softmax_cross_entropy"]
