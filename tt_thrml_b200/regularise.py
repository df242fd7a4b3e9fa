"""Dropout of units by a counter-based generator.

    y[i] = keep[i] * x[i] / (1 - p),   keep[i] = (16 bits of Philox4x32-10) >= round(65536 p)

The bits of element i come from draw i // 8 of (seed, step), so the mask depends
on neither the launch nor the device and is never stored: the backward pass draws
it again.  The probability that applies is round(65536 p) / 65536, and the factor
goes with it, so means are kept exactly.
"""

from __future__ import annotations

from . import _native as nat
from .quantized import dtype_code, on_device, require_cuda


def _torch():
    import torch

    return torch


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
    with on_device(x.device):
        return nat.bound_hostcall().dropout(x, round(65536 * p), seed, step, step_at)


__all__ = ["dropout"]
