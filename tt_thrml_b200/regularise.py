"""Dropout of units by a counter-based generator.

    y[i] = keep[i] * x[i] / (1 - p),   keep[i] = (16 bits of Philox4x32-10) >= round(65536 p)

The bits of element i come from draw i // 8 of (seed, step), so the mask depends
on neither the launch nor the device and is never stored: the backward pass draws
it again.  The probability that applies is round(65536 p) / 65536, and the factor
goes with it, so means are kept exactly.
"""

from __future__ import annotations

from . import _native as nat
from .quantized import dtype_code, on_device, raw_stream, require_cuda

_function = None


def _torch():
    import torch

    return torch


def _launch(x, cut, seed, step, step_at, used):
    torch = _torch()
    x = x.contiguous()
    y = torch.empty_like(x)
    if x.numel():
        with on_device(x.device):
            nat.check(
                nat.lib().tthrml_dropout(x.data_ptr(), dtype_code(x.dtype), x.numel(), cut, seed, step, nat.ptr(step_at),
                                         1 if step_at is not None and step_at.dtype == torch.int64 else 0, nat.ptr(used),
                                         y.data_ptr(), raw_stream(x.device.index)),
                "tthrml_dropout",
            )
    return y


def _autograd_function():
    global _function
    if _function is not None:
        return _function
    torch = _torch()

    class Dropout(torch.autograd.Function):
        @staticmethod
        def forward(ctx, x, cut, seed, step, step_at):
            # a step on the device may have moved on by the time of the backward pass: the kernel leaves what it used
            used = None if step_at is None else torch.empty(1, dtype=torch.int32, device=x.device)
            ctx.draws = (cut, seed, step)
            ctx.save_for_backward(used if x.numel() else None)
            return _launch(x, cut, seed, step, step_at, used)

        @staticmethod
        def backward(ctx, grad):
            (used,) = ctx.saved_tensors
            return Dropout.apply(grad, *ctx.draws, used), None, None, None, None

    _function = Dropout
    return _function


def dropout(x, p=0.5, *, seed, step=0):
    """x with elements set to 0 with probability p and the others scaled to keep the mean; differentiable in x (any number
    of times).

    x: float32, bfloat16 or float16, any shape and strides; the element of position i
    in row-major order takes the i-th 16 bits.  seed: 0 to 2^64 - 1.  step: which of
    the seed's masks, 0 to 2^32 - 1, or an int32 / int64 tensor of one element on
    x's device that the kernel reads (a captured graph then takes another mask each
    time it is replayed after the step was changed).  Dropped elements are 0 even
    where x is infinite or NaN.  Launched on the current stream of x's device.
    """
    torch = _torch()
    require_cuda("x", x)
    if dtype_code(x.dtype) is None:
        raise ValueError(f"x must be float32, bfloat16 or float16, got {x.dtype}")
    p = float(p)
    if not 0.0 <= p <= 1.0:
        raise ValueError(f"p must be between 0 and 1, got {p}")
    seed = int(seed)
    if not 0 <= seed < 2**64:
        raise ValueError(f"seed must be between 0 and 2^64 - 1, got {seed}")
    step_at = None
    if isinstance(step, torch.Tensor):
        require_cuda("step", step, x.device)
        if step.dtype not in (torch.int32, torch.int64) or step.numel() != 1:
            raise ValueError(f"step must be one int32 or int64, got {step.dtype} of shape {tuple(step.shape)}")
        step, step_at = 0, step
    else:
        step = int(step)
        if not 0 <= step < 2**32:
            raise ValueError(f"step must be between 0 and 2^32 - 1, got {step}")
    return _autograd_function().apply(x, round(65536 * p), seed, step, step_at)


__all__ = ["dropout"]
