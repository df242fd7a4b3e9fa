"""Softmax cross entropy of categories that are read out of a block's units.

    l[t, v] = sum_k x[t, k] w[v, k] + bias[v],   loss[t] = log sum_v exp l[t, v] - l[t, y[t]]

The logits are never held as a whole: the forward pass keeps a running maximum
and sum per row, the backward pass takes the categories in pieces (at most
256 MiB of 16-bit differences exp(l - z) - [v = y] at a time).  x is a dense
block's units over the chains (or any features), w one row per category.

The kernels launch on the current stream of x's device; nothing synchronises.
A kernel whose wait expires (two seconds) gives up and leaves a code that
check_operator_errors reports.
"""

from __future__ import annotations

from . import _native as nat
from .moments import _lay_out
from .quantized import dtype_code, error_word, on_device, raw_stream, require_cuda

_REDUCTIONS = {"none": 0, "mean": 1, "sum": 2}
_function = None


def _torch():
    import torch

    return torch


class _Call:
    """What the passes over one batch share: the problem as the library takes it, and what it points to."""

    def __init__(self, x, weights, targets, bias, ignored, stream):
        torch = _torch()
        dev = x.device
        laid, held = _lay_out([x, weights], dev, stream)
        bias = None if bias is None else bias.contiguous()
        targets = targets.contiguous()
        self.held = (x, weights, targets, bias, held)
        p = self.problem = nat.Xent()
        p.x, p.x_ld = laid[0]
        p.w, p.w_ld = laid[1]
        p.targets = targets.data_ptr()
        p.bias = None if bias is None else bias.data_ptr()
        p.rows, p.cols = x.shape
        p.categories = weights.shape[0]
        p.ignored = ignored
        p.dtype = dtype_code(x.dtype)
        p.wide_targets = 1 if targets.dtype == torch.int64 else 0


def _workspace(size: int, dev, what: str):
    torch = _torch()
    if size < 0:
        nat.check(size, what)
    return torch.empty(max(size, 16), dtype=torch.uint8, device=dev), size


def _forward(call, reduction):
    """(losses of the rows, (reduced loss, 1 / rows that count) or None, log2 of the normalisers)."""
    torch = _torch()
    p, dev = call.problem, call.held[0].device
    lib = nat.lib()
    space, size = _workspace(lib.tthrml_xent_forward_workspace(p.rows, p.categories), dev, "tthrml_xent_forward_workspace")
    rows = torch.empty((2, p.rows), dtype=torch.float32, device=dev)
    reduced = torch.empty(2, dtype=torch.float32, device=dev) if reduction else None
    nat.check(
        lib.tthrml_xent_forward(p, rows[0].data_ptr(), rows[1].data_ptr(), nat.ptr(reduced), reduction, space.data_ptr(), size,
                                error_word(dev).data_ptr(), raw_stream(dev.index)),
        "tthrml_xent_forward",
    )
    return rows[1], reduced, rows[0]


def backward(call, log2_z, grad, inv_count, dx, dw, db) -> None:
    """Gradients of sum_t weight_t loss_t into dx, dw (one type, dense rows) and db, each a tensor or None.  The weights are
    grad * inv_count (one element each, inv_count may be None), or grad's elements, one per row."""
    p, dev = call.problem, call.held[0].device
    lib = nat.lib()
    space, size = _workspace(
        lib.tthrml_xent_backward_workspace(p.rows, p.categories, p.cols, dx is not None, dw is not None, db is not None), dev,
        "tthrml_xent_backward_workspace")
    code = dtype_code(next((t.dtype for t in (dx, dw) if t is not None), call.held[0].dtype))
    nat.check(
        lib.tthrml_xent_backward(p, log2_z.data_ptr(), grad.data_ptr(), 1 if grad.dim() else 0, nat.ptr(inv_count), nat.ptr(dx),
                                 p.cols, nat.ptr(dw), p.cols, code, nat.ptr(db), space.data_ptr(), size,
                                 error_word(dev).data_ptr(), raw_stream(dev.index)),
        "tthrml_xent_backward",
    )


def _autograd_function():
    global _function
    if _function is not None:
        return _function
    torch = _torch()

    class SoftmaxCrossEntropy(torch.autograd.Function):
        @staticmethod
        def forward(ctx, x, weights, bias, targets, reduction, ignored):
            with on_device(x.device):
                call = _Call(x, weights, targets, bias, ignored, raw_stream(x.device.index))
                rows, reduced, log2_z = _forward(call, reduction)
            ctx.call, ctx.reduction = call, reduction
            # the tensors themselves, so that a change in place before the backward pass is noticed
            ctx.save_for_backward(x, weights, bias, targets, log2_z, reduced)
            return rows if reduction == 0 else reduced[0]

        @staticmethod
        @torch.autograd.function.once_differentiable
        def backward(ctx, grad):
            x, weights, bias, _, log2_z, reduced = ctx.saved_tensors
            need_x, need_w, need_b = ctx.needs_input_grad[:3]
            dx = torch.empty(x.shape, dtype=x.dtype, device=x.device) if need_x else None
            dw = torch.empty(weights.shape, dtype=weights.dtype, device=x.device) if need_w else None
            db = torch.empty(bias.shape, dtype=bias.dtype, device=x.device) if need_b else None
            with on_device(x.device):
                backward(ctx.call, log2_z, grad.contiguous(), None if reduced is None else reduced[1], dx, dw, db)
            return dx, dw, db, None, None, None

    _function = SoftmaxCrossEntropy
    return _function


def softmax_cross_entropy(x, weights, targets, *, bias=None, reduction="mean", ignore_index=-100):
    """Minus the log likelihood of the target categories under softmax(x weights^T + bias), differentiable in x, weights
    and bias.

    x: bfloat16 or float16 [..., K]; weights: the same type [V, K], any strides
    (rows that are not 16-byte aligned are laid out again in each call); targets:
    int64 or int32 [...]; bias: float32 [V], -inf for categories that cannot occur.
    reduction "mean" (over the rows that count), "sum" (float32 scalars) or "none"
    (float32 [...]).  Rows whose target is `ignore_index` do not count: loss 0, no
    gradient (their values must be finite, as 0 times them is added to the weights'
    gradient); a mean over no rows is 0.  A target outside 0 .. V - 1 gives NaN.  A
    row in which no category can occur has loss inf and no gradient.

    Sums and normalisers are float32; the gradients are products of 16-bit
    differences, accumulated in float32.  The result is the same every time.
    Gradients of gradients and forward-mode derivatives are not available.
    """
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
    if reduction not in _REDUCTIONS:
        raise ValueError(f"reduction must be 'mean', 'sum' or 'none', got {reduction!r}")
    lead = x.shape[:-1]
    rows = targets.numel()
    if rows > nat.XENT_MAX_ROWS:
        raise ValueError(f"at most {nat.XENT_MAX_ROWS} rows are supported, got {rows}")
    if rows == 0:  # nothing counts
        zero = x.sum(-1).float() + weights[:0].sum().float() + (0.0 if bias is None else bias[:0].sum())
        return zero if reduction == "none" else zero.sum()
    error_word(dev)  # made before the first capture
    flat = x.reshape(rows, K)
    loss = _autograd_function().apply(flat, weights, bias, targets.reshape(rows), _REDUCTIONS[reduction], int(ignore_index))
    return loss.reshape(lead) if reduction == "none" else loss


__all__ = ["softmax_cross_entropy"]
