"""Pair moments of two blocks over the chain batch: what a dense program's couplings are learned from.

    out[i, j] = sum_p s_p sum_c x_p[c, i] y_p[c, j]

over one or several phases p (data against model), with the unit sums
sum_p s_p sum_c x_p[c, i].  The observers accumulate listed products of a
row-major state (`DeviceMomentObserver`); this is the same for every pair of
two dense blocks at once, on the tensor cores.
"""

from __future__ import annotations

from . import _native as nat
from .quantized import (
    _error_addresses,
    current_device,
    dtype_code,
    error_word,
    mark_written,
    on_device,
    raw_stream,
    refuse_grad,
    refuse_overlap,
    refuse_shared_outputs,
    refuse_written_grad,
    require_cuda,
)


def _torch():
    import torch

    return torch


def _lay_out(tensors, dev, stream):
    """[(address, pitch)] of chain-major operands as the kernel reads them, rows 16-byte aligned; the others are
    copied into one buffer by one launch, which is returned too (it must live until the kernel is queued)."""
    torch = _torch()
    found, again, size = [], [], 0
    for i, t in enumerate(tensors):
        rows, units = t.shape
        ld = t.stride(0) if rows > 1 else -(-units // 8) * 8
        if (units == 1 or t.stride(1) == 1) and ld % 8 == 0 and ld >= units and t.data_ptr() % 16 == 0:
            found.append((t.data_ptr(), ld))
            continue
        pitch = -(-units // 8) * 8
        again.append((i, t, pitch, size))
        found.append(None)
        size += rows * pitch
    if not again:
        return found, None
    buffer = torch.empty(max(size, 8), dtype=tensors[0].dtype, device=dev)
    rows = (nat.PackMatrix * len(again))()
    for row, (i, t, pitch, at) in zip(rows, again):
        row.src, row.dst, row.pitch = t.data_ptr(), buffer.data_ptr() + 2 * at, pitch
        row.rows, row.cols = t.shape
        row.row_stride, row.col_stride = t.stride()
        found[i] = (row.dst, pitch)
    nat.check(nat.lib().tthrml_pack_rows(rows, len(again), stream), "tthrml_pack_rows")
    return found, buffer


def _sum_target(name, t, n, dev):
    torch = _torch()
    require_cuda(name, t, dev)
    if t.dtype != torch.float32 or tuple(t.shape) != (n,) or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous float32 tensor of shape ({n},), got {t.dtype} of {tuple(t.shape)}")
    return t


def pair_moments(x, y, scale=1.0, *, out=None, accumulate=False, units=False):
    """sum_p scale_p x_p^T y_p in float32 [M, N]; with `units` also sum_p scale_p x_p.sum(0) and the same of y.

    x, y: one tensor each ([chains, M] and [chains, N], bfloat16 or float16,
    one type) or sequences of them, one per phase (at most 6; chains may differ
    between phases and may be 0); scale: a number or one per phase.  out: float32
    [M, N] with dense rows (with `units` a tuple of out, x_sum [M], y_sum [N]) to
    write, or, with `accumulate`, to add to.  The result is the same every time.
    An in-kernel wait that expires is reported by check_operator_errors().
    """
    torch = _torch()
    xs, ys = ([t] if isinstance(t, torch.Tensor) else list(t) for t in (x, y))
    scales = [float(scale)] * len(xs) if isinstance(scale, (int, float)) else [float(s) for s in scale]
    if not xs or not len(xs) == len(ys) == len(scales):
        raise ValueError(f"x, y and scale need one entry per phase, got {len(xs)}, {len(ys)} and {len(scales)}")
    if len(xs) > nat.MAX_PHASES:
        raise ValueError(f"at most {nat.MAX_PHASES} phases are supported, got {len(xs)}")
    if out is None and not accumulate and type(xs[0]) is torch.Tensor:
        index = xs[0].get_device()
        word = _error_addresses.get(index)
        if word is not None and current_device() == index:  # the plain case, from the second call on
            nat.bind_device(index)
            made = nat.hostcall().pair_moments(xs, ys, scales, bool(units), nat.address_of("tthrml_pair_moments"),
                                               nat.address_of("tthrml_pair_moments_packed"), word, raw_stream(index), index)
            if made is not None:
                if type(made) is int:
                    nat.check(made, "tthrml_pair_moments")
                return made
    require_cuda("x", xs[0])
    dev, dtype = xs[0].device, xs[0].dtype
    code = dtype_code(dtype)
    if code not in (nat.DT_BF16, nat.DT_F16):
        raise ValueError(f"x and y must be bfloat16 or float16, got {dtype}")
    shapes = []
    for p, (a, b) in enumerate(zip(xs, ys)):
        for name, t in (("x", a), ("y", b)):
            require_cuda(name, t, dev)
            if t.dtype != dtype or t.dim() != 2:
                raise ValueError(f"{name}[{p}] must be a {dtype} matrix, got {t.dtype} of shape {tuple(t.shape)}")
            refuse_grad(f"{name}[{p}]", t, "pair moments")
        (chains, m), (other, n) = a.shape, b.shape
        if chains != other:
            raise ValueError(f"phase {p}: x has {chains} chains, y has {other}")
        shapes.append((m, n))
    if shapes.count(shapes[0]) != len(shapes):
        raise ValueError(f"every phase needs the same units, got {shapes}")
    M, N = shapes[0]
    if M < 1 or N < 1:
        raise ValueError(f"both blocks need units, got {M} and {N}")
    x_sum = y_sum = None
    if out is None:
        if accumulate:
            raise ValueError("accumulate needs out")
        out = torch.empty((M, N), dtype=torch.float32, device=dev)
        if units:
            x_sum, y_sum = (torch.empty(n, dtype=torch.float32, device=dev) for n in (M, N))
    else:
        if units:
            out, x_sum, y_sum = out
            _sum_target("x_sum", x_sum, M, dev)
            _sum_target("y_sum", y_sum, N, dev)
        require_cuda("out", out, dev)
        if out.dtype != torch.float32 or tuple(out.shape) != (M, N):
            raise ValueError(f"out must be float32 of shape {(M, N)}, got {out.dtype} of {tuple(out.shape)}")
        if (N > 1 and out.stride(1) != 1) or (M > 1 and out.stride(0) < N):
            raise ValueError("out needs dense rows that do not overlap")
        inputs = [(f"{name}[{p}]", t) for name, ts in (("x", xs), ("y", ys)) for p, t in enumerate(ts)]
        outs = [(name, t) for name, t in (("out", out), ("x_sum", x_sum), ("y_sum", y_sum)) if t is not None]
        refuse_shared_outputs(outs)
        for name, t in outs:
            refuse_overlap(name, t, inputs)
            refuse_written_grad(name, t)
        mark_written(*(t for _, t in outs))
    phases = (nat.MomentPhase * len(xs))()
    with on_device(dev):
        stream = raw_stream(dev.index)
        laid, held = _lay_out(xs + ys, dev, stream)
        for p, (row, s) in enumerate(zip(phases, scales)):
            row.x, row.x_ld = laid[p]
            row.y, row.y_ld = laid[len(xs) + p]
            row.chains = xs[p].shape[0]
            row.scale = row.x_scale = row.y_scale = s
        launch(phases, code, M, N, out, x_sum, y_sum, accumulate, dev, stream)
    del held
    return (out, x_sum, y_sum) if units else out


def launch(phases, code, M, N, out, x_sum, y_sum, accumulate, dev, stream) -> None:
    """tthrml_pair_moments on a cudaStream_t of `dev`."""
    nat.check(
        nat.lib().tthrml_pair_moments(
            phases, len(phases), code, M, N, out.data_ptr(), out.stride(0) if M > 1 else N,
            None if x_sum is None else x_sum.data_ptr(), None if y_sum is None else y_sum.data_ptr(),
            1 if accumulate else 0, error_word(dev).data_ptr(), stream,
        ),
        "tthrml_pair_moments",
    )


__all__ = ["pair_moments"]
