"""8-bit integer products: fields of a batch of rows through weights held as int8.

    y[m, n] = (sum_k q[m, k] w[n, k]) * (s_x[m] * s_w[n]) + bias[n]

with one float32 scale per row m (token / chain) and per unit n (channel).
`quantize_rows` makes the integers and scales of a matrix, `QuantizedRows`
holds them, `int8_product` multiplies; rows given as floats are quantised
within the call.  The sums are exact in int32, so the result does not depend
on how the kernels split them.  A dense program runs its sweeps on the same
arithmetic with `dense_precision="int8"` (make_cuda_config).

The kernels launch on the current stream of the rows' device; nothing
synchronises.  A kernel whose wait for its own copies or products expires (two
seconds) gives up and leaves a code that check_operator_errors reports.
There is no backward pass and no forward-mode derivative: rows, biases and
scales that require a gradient or carry a tangent are refused.
"""

from __future__ import annotations

import contextlib

from . import _native as nat


def _torch():
    import torch

    return torch


_codes: dict = {}


def dtype_code(dtype):
    """The C ABI's code of a floating element type, or None."""
    if not _codes:
        torch = _torch()
        _codes.update({torch.float32: nat.DT_F32, torch.bfloat16: nat.DT_BF16, torch.float16: nat.DT_F16})
    return _codes.get(dtype)


def current_device() -> int:
    torch = _torch()
    return torch._C._cuda_getDevice()


def raw_stream(index: int) -> int:
    """The current stream of a device as a cudaStream_t."""
    torch = _torch()
    return torch._C._cuda_getCurrentRawStream(index)


_error_words: dict = {}
_error_addresses: dict = {}


def error_word(device):
    """The device's int32 word that operator kernels set when an in-kernel wait expires."""
    word = _error_words.get(device.index)
    if word is None:
        torch = _torch()
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError("run the operator once on this device before capturing it into a CUDA graph")
        word = _error_words[device.index] = torch.zeros(1, dtype=torch.int32, device=device)
        torch.cuda.current_stream(device).synchronize()
        _error_addresses[device.index] = word.data_ptr()
    return word


def check_operator_errors(device=None) -> None:
    """Raises if an operator kernel on `device` (default: every device used) reported an expired wait since the last
    report; what such a kernel wrote is not its result.  Synchronises."""
    torch = _torch()
    found = []
    for index, word in list(_error_words.items()):
        if device is not None and torch.device(device).index not in (None, index):
            continue
        torch.cuda.synchronize(index)
        code = int(word.item())
        if code:
            found.append(f"a device kernel reported an expired wait (code {code}, device {index})")
            word.zero_()  # reported once
            torch.cuda.synchronize(index)
    if found:
        raise RuntimeError("; ".join(found))


@contextlib.contextmanager
def _other_device(index: int):
    torch = _torch()
    with torch.cuda.device(index):
        nat.check(nat.lib().tthrml_set_device(index), "tthrml_set_device")
        nat._bound.device = index
        try:
            yield
        finally:
            nat._bound.device = None  # the library's current device follows torch's again at the next call


def on_device(device):
    """Context in which `device` is current for torch and for the library; cheap when it already is."""
    torch = _torch()
    if torch.cuda.current_device() != device.index:
        return _other_device(device.index)
    nat.bind_device(device.index)
    return contextlib.nullcontext()


def require_cuda(name: str, t, device=None):
    torch = _torch()
    if isinstance(t, torch.Tensor) and t.is_cuda and (device is None or t.device == device):
        return
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a torch tensor, got {type(t).__name__}")
    if not t.is_cuda:
        raise ValueError(f"{name} must be on a CUDA device (there is no CPU path), got {t.device}")
    raise ValueError(f"{name} is on {t.device}, expected {device}")


def refuse_grad(name: str, t, what: str) -> None:
    """Raises for an input whose derivative `what`, which have none, would drop: a gradient asked for, or the tangent
    of a forward-mode dual tensor."""
    torch = _torch()
    if torch.is_grad_enabled() and t.requires_grad:
        raise RuntimeError(f"{name} requires a gradient, but {what} have no backward pass (use torch.no_grad())")
    if torch.autograd.forward_ad.unpack_dual(t).tangent is not None:
        raise RuntimeError(f"{name} carries a tangent, but {what} have no forward-mode derivative")


def _no_grad(name: str, t):
    refuse_grad(name, t, "8-bit products")


def refuse_written_grad(name: str, out) -> None:
    """Raises for an output that requires a gradient: kernels write it behind autograd's back."""
    torch = _torch()
    if torch.is_grad_enabled() and out.requires_grad:
        raise RuntimeError(f"{name} requires a gradient and cannot be written in place (use torch.no_grad())")


def mark_written(*outs) -> None:
    """Tells autograd that a kernel wrote the tensors: backward passes that saved them raise."""
    nat.hostcall().bump_versions(list(outs))


def memory_span(t) -> tuple[int, int]:
    """First and last-plus-one address that a tensor's elements lie in."""
    if not t.numel():
        return 0, 0
    reach = sum((n - 1) * st for n, st in zip(t.shape, t.stride())) + 1
    return t.data_ptr(), t.data_ptr() + reach * t.element_size()


def _memory_rows(t) -> tuple[int, int] | None:
    """(bytes from row to row, bytes of a row) of a tensor whose rows are dense and equally far apart, else None; one row
    is as far from the next as any other tensor's."""
    dims = [(n, st) for n, st in zip(t.shape, t.stride()) if n != 1]
    width = 1
    if dims and dims[-1][1] == 1:
        width = dims.pop()[0]
    if not dims:
        return 0, width * t.element_size()
    pitch = dims[-1][1]
    if any(a[1] != b[0] * b[1] for a, b in zip(dims, dims[1:])):
        return None
    return pitch * t.element_size(), width * t.element_size()


def share_memory(t, u) -> bool:
    """Whether two tensors may share memory: their spans meet, and they are not two ranges of columns of one matrix."""
    (a, b), (c, d) = memory_span(t), memory_span(u)
    if not (a < d and c < b):
        return False
    rows, other = _memory_rows(t), _memory_rows(u)
    if rows is None or other is None:
        return True
    pitch = rows[0] or other[0]
    if pitch == 0 or (other[0] or pitch) != pitch:
        return True
    gap = (c - a) % pitch  # from a row of t to the next start of one of u
    return not (rows[1] <= gap and gap + other[1] <= pitch)


def refuse_overlap(name: str, out, inputs) -> None:
    for other, t in inputs:
        if share_memory(out, t):
            raise ValueError(f"{name} shares memory with {other}, which the kernel reads meanwhile")


def refuse_shared_outputs(outs) -> None:
    """Raises if two of the (name, tensor) outputs of one call share memory: the kernel writes both."""
    for i, (name, t) in enumerate(outs):
        for other, u in outs[i + 1 :]:
            if share_memory(t, u):
                raise ValueError(f"{name} and {other} share memory, and the kernel writes both")


class QuantizedRows:
    """A matrix as int8 rows with one float32 scale per row: value[r, c] = values[r, c] * scale[r].

    values: int8 [rows, cols]; rows that are not 16-byte aligned and a
    multiple of 16 bytes apart are laid out again once, here.  scale: float32
    [rows], or None for ones (spins as +-1 are their own integers).
    """

    def __init__(self, values, scale=None):
        torch = _torch()
        require_cuda("values", values)
        if values.dtype != torch.int8 or values.dim() != 2:
            raise ValueError(f"values must be an int8 matrix, got {values.dtype} of shape {tuple(values.shape)}")
        rows, cols = values.shape
        if cols < 1 or cols > nat.INT8_MAX_COLS:
            raise ValueError(f"1 to {nat.INT8_MAX_COLS} columns are supported, got {cols}")
        if scale is not None:
            require_cuda("scale", scale, values.device)
            if scale.dtype != torch.float32 or scale.dim() != 1 or scale.shape[0] != rows:
                raise ValueError(f"scale must be float32 of shape ({rows},), got {scale.dtype} of {tuple(scale.shape)}")
            scale = scale.contiguous()
        pitch = values.stride(0) if rows > 1 else -(-cols // 16) * 16
        if (cols > 1 and values.stride(1) != 1) or pitch % 16 or pitch < cols or values.data_ptr() % 16:
            laid = torch.empty((rows, -(-cols // 16) * 16), dtype=torch.int8, device=values.device)
            laid[:, :cols].copy_(values)
            values = laid[:, :cols]
            pitch = laid.shape[1]
        self.values = values
        self.index = values.device.index
        self.scale = scale
        self.pitch = int(pitch)

    @property
    def shape(self):
        return self.values.shape

    @property
    def device(self):
        return self.values.device

    def dequantize(self):
        """The float32 matrix that the integers and scales stand for."""
        v = self.values.float()
        return v if self.scale is None else v * self.scale[:, None]


def quantize_rows(x) -> QuantizedRows:
    """Rows of a float32, bfloat16 or float16 matrix as int8 with one scale per row.

    scale[r] = max|x_r| / 127 and q = rint(x 127 / max|x_r|), both in float32.
    A row of zeros (or of magnitudes below 2^-120) gets scale 0, a row that
    holds an infinity or NaN gets scale NaN.  Any strides; rows and transposed
    matrices are read at full width.
    """
    torch = _torch()
    require_cuda("x", x)
    code = dtype_code(x.dtype)
    if code is None or x.dim() != 2:
        raise ValueError(f"x must be a float32, bfloat16 or float16 matrix, got {x.dtype} of shape {tuple(x.shape)}")
    _no_grad("x", x)
    rows, cols = x.shape
    if cols < 1 or cols > nat.INT8_MAX_COLS:
        raise ValueError(f"1 to {nat.INT8_MAX_COLS} columns are supported, got {cols}")
    if x.stride(1) == 0 and cols > 1:
        x = x.contiguous()
    pitch = -(-cols // 16) * 16
    values = torch.empty((rows, pitch), dtype=torch.int8, device=x.device)
    scale = torch.empty(rows, dtype=torch.float32, device=x.device)
    if rows:
        with on_device(x.device):
            nat.check(
                nat.lib().tthrml_quantize_rows(
                    x.data_ptr(), code, rows, cols, x.stride(0), x.stride(1) if cols > 1 else 1, values.data_ptr(),
                    pitch, scale.data_ptr(), raw_stream(x.device.index),
                ),
                "tthrml_quantize_rows",
            )
    return QuantizedRows(values[:, :cols], scale)


def int8_product(x, weights: QuantizedRows, *, bias=None, out_dtype=None, out=None):
    """y = x w^T with 8-bit integers: x [..., K] (float rows, quantised here, or QuantizedRows), weights [N, K].

    bias: float32 [N] added after the scaling.  out_dtype: float32, bfloat16
    or float16 (default: x's type; float32 for QuantizedRows).  out: a tensor
    [..., N] to write, its rows dense.  One or two rows run as one launch that
    reads the weights once; more rows are quantised and multiplied on the
    tensor cores.
    """
    if out is None and out_dtype is None and type(weights) is QuantizedRows and weights.scale is not None:
        index = weights.index
        word = _error_addresses.get(index)
        if word is not None and current_device() == index:  # the plain case, from the second call on
            nat.bind_device(index)
            y = nat.hostcall().int8_product(x, weights.values, weights.scale, weights.pitch, bias,
                                            nat.address_of("tthrml_int8_linear"), word, raw_stream(index), index)
            if y is not None:
                if type(y) is int:
                    nat.check(y, "tthrml_int8_linear")
                return y
    torch = _torch()
    if not isinstance(weights, QuantizedRows):
        raise TypeError(f"weights must be QuantizedRows (see quantize_rows), got {type(weights).__name__}")
    w, w_scale = weights.values, weights.scale
    if w_scale is None:
        raise ValueError("weights need a scale per unit")
    dev, N = w.device, w.shape[0]
    quantized = isinstance(x, QuantizedRows)
    rows = x.values if quantized else x
    require_cuda("x", rows, dev)
    code = nat.DT_I8 if quantized else dtype_code(x.dtype)
    if code is None or rows.dim() < 1:
        raise ValueError(f"x must hold float32, bfloat16 or float16 rows, got {x.dtype} of shape {tuple(x.shape)}")
    _no_grad("x", rows)
    for name, q in (("x", x), ("weights", weights)):
        if isinstance(q, QuantizedRows) and q.scale is not None:
            _no_grad(f"the scale of {name}", q.scale)
    lead, K = rows.shape[:-1], rows.shape[-1]
    if K != w.shape[1]:
        raise ValueError(f"x has rows of {K}, the weights have {w.shape[1]} columns")
    bias_at = None
    if bias is not None:
        require_cuda("bias", bias, dev)
        if bias.dtype != torch.float32 or bias.shape != (N,):
            raise ValueError(f"bias must be float32 of shape ({N},), got {bias.dtype} of {tuple(bias.shape)}")
        _no_grad("bias", bias)
        bias = bias.contiguous()
        bias_at = bias.data_ptr()
    if out_dtype is None:
        out_dtype = out.dtype if out is not None else (torch.float32 if quantized else x.dtype)
    out_code = dtype_code(out_dtype)
    if out_code is None:
        raise ValueError(f"out_dtype must be float32, bfloat16 or float16, got {out_dtype}")
    given = out is not None
    if not given:
        out, out_ld = torch.empty((*lead, N), dtype=out_dtype, device=dev), N
    else:
        require_cuda("out", out, dev)
        if out.dtype != out_dtype or out.shape != (*lead, N):
            raise ValueError(f"out must be {out_dtype} of shape {(*lead, N)}, got {out.dtype} of {tuple(out.shape)}")
        refuse_written_grad("out", out)
        flat = out.view(-1, N) if N else out  # raises if the rows cannot be one matrix
        if flat.numel() and ((N > 1 and flat.stride(1) != 1) or (flat.shape[0] > 1 and flat.stride(0) < N)):
            raise ValueError("out needs dense rows that do not overlap")
        inputs = [("x", rows), ("the weights", w), ("the weights' scales", w_scale)]
        refuse_overlap("out", out, inputs + ([] if bias is None else [("bias", bias)]))
        out_ld = flat.stride(0) if N and flat.shape[0] > 1 else N
    if not out.numel():
        return out
    if given:
        mark_written(out)
    if rows.dim() != 2:
        rows = rows.reshape(-1, K)
    M = rows.shape[0]
    row_stride, col_stride = rows.stride()
    index = dev.index
    lib = nat.lib()
    with on_device(dev):
        stream = raw_stream(index)
        error = error_word(dev).data_ptr()
        if not quantized:
            if K == 1:
                col_stride = 1
            elif col_stride == 0:
                rows = rows.contiguous()
                row_stride, col_stride = rows.stride()
            pitch = -(-K // 16) * 16
            workspace, size = None, 0
            if M > 2 or M * pitch > nat.INT8_FEW_BYTES or col_stride != 1 or (M > 1 and row_stride < K):
                size = M * pitch + -(-M // 4) * 16
                workspace = torch.empty(size, dtype=torch.int8, device=dev)
            rc = lib.tthrml_int8_linear(
                rows.data_ptr(), code, M, K, row_stride, col_stride, None if workspace is None else workspace.data_ptr(),
                size, w.data_ptr(), weights.pitch, w_scale.data_ptr(), N, bias_at, out.data_ptr(), out_code, out_ld, error,
                stream,
            )
            nat.check(rc, "tthrml_int8_linear")
            return out
        x_scale = None if x.scale is None else x.scale.data_ptr()
        if M <= 2 and M * (-(-K // 16) * 16) <= nat.INT8_FEW_BYTES:
            rc = lib.tthrml_int8_product_few(
                rows.data_ptr(), code, x.pitch, x_scale, w.data_ptr(), weights.pitch, w_scale.data_ptr(), M, N, K,
                bias_at, out.data_ptr(), out_code, out_ld, stream,
            )
            nat.check(rc, "tthrml_int8_product_few")
            return out
        rc = lib.tthrml_int8_product(
            rows.data_ptr(), x.pitch, x_scale, w.data_ptr(), weights.pitch, w_scale.data_ptr(), M, N, K, bias_at,
            out.data_ptr(), out_code, out_ld, error, stream,
        )
        nat.check(rc, "tthrml_int8_product")
    return out


__all__ = ["QuantizedRows", "quantize_rows", "int8_product", "check_operator_errors"]
