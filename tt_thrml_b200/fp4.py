"""4-bit floating point products: fields of a batch of rows through weights held in 4 bits.

    value[r, c] = code[r, c] * block[r, c // 16] * scale[r]
    y[m, n] = (sum_k x[m, k] w[n, k]) + bias[n]

with codes e2m1 (0, 1/2, 1, 3/2, 2, 3, 4, 6 and their negatives), a scale e4m3
per 16 columns and a float32 scale per row (token / chain, unit / channel).
`quantize_fp4` makes them from a matrix, `Fp4Rows` holds them, `fp4_product`
multiplies on the tensor cores at four times the rate of 16-bit operands; rows
given as floats are quantised within the call.  A spin of +-1 is its own code.

The kernels launch on the current stream of the rows' device; nothing
synchronises.  A kernel whose wait for its own copies or products expires (two
seconds) gives up and leaves a code that check_operator_errors reports.
There is no backward pass and no forward-mode derivative: rows, biases and
scales that require a gradient or carry a tangent are refused.
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
    refuse_written_grad,
    require_cuda,
)

BLOCK = 16  # columns that share a block scale


def _torch():
    import torch

    return torch


def _no_grad(name: str, t):
    refuse_grad(name, t, "4-bit products")


def _scale_bytes(rows: int, cols: int) -> int:
    return -(-rows // 128) * -(-cols // 256) * 2048


def _check_cols(cols: int) -> None:
    if cols < 1 or cols > nat.FP4_MAX_COLS:
        raise ValueError(f"1 to {nat.FP4_MAX_COLS} columns are supported, got {cols}")


class Fp4Rows:
    """A matrix of 4-bit values with a scale per 16 columns and one per row.

    codes: uint8 [rows, ceil(cols / 2)], two codes to a byte, the even column in
    the low half.  block_scale: float8_e4m3fn [rows, ceil(cols / 16)], not
    negative.  scale: float32 [rows].  cols: the columns (default: two per byte).
    Codes whose rows are not 16-byte aligned and a multiple of 16 bytes apart, or of
    odd columns (the half byte behind the last one is not read), and the block
    scales, are laid out again once, here.
    """

    def __init__(self, codes, block_scale, scale, *, cols=None):
        torch = _torch()
        require_cuda("codes", codes)
        if codes.dtype != torch.uint8 or codes.dim() != 2:
            raise ValueError(f"codes must be a uint8 matrix, got {codes.dtype} of shape {tuple(codes.shape)}")
        rows, bytes_ = codes.shape
        cols = 2 * bytes_ if cols is None else int(cols)
        _check_cols(cols)
        if bytes_ != -(-cols // 2):
            raise ValueError(f"{cols} columns are {-(-cols // 2)} bytes of codes, got {bytes_}")
        require_cuda("block_scale", block_scale, codes.device)
        blocks = -(-cols // BLOCK)
        if block_scale.dtype != torch.float8_e4m3fn or tuple(block_scale.shape) != (rows, blocks):
            raise ValueError(f"block_scale must be float8_e4m3fn of shape {(rows, blocks)}, got {block_scale.dtype} of "
                             f"{tuple(block_scale.shape)}")
        require_cuda("scale", scale, codes.device)
        if scale.dtype != torch.float32 or tuple(scale.shape) != (rows,):
            raise ValueError(f"scale must be float32 of shape ({rows},), got {scale.dtype} of {tuple(scale.shape)}")
        pitch = codes.stride(0) if rows > 1 else -(-bytes_ // 16) * 16
        if cols % 2 or (bytes_ > 1 and codes.stride(1) != 1) or pitch % 16 or pitch < bytes_ or codes.data_ptr() % 16:
            laid = torch.zeros((rows, -(-bytes_ // 16) * 16), dtype=torch.uint8, device=codes.device)
            laid[:, :bytes_].copy_(codes)
            if cols % 2:
                laid[:, bytes_ - 1] &= 15  # the half behind the last column counts in no product
            codes, pitch = laid[:, :bytes_], laid.shape[1]
        # [row block, 4 x 32 rows, column block, 4 x 4 scales] -> [row block, column block, 4, 32 rows, 4 row groups, 4]
        m, k = -(-rows // 128), -(-cols // 256)
        padded = torch.zeros((m * 128, k * 16), dtype=torch.uint8, device=codes.device)
        padded[:rows, :blocks].copy_(block_scale.view(torch.uint8))
        laid = padded.view(m, 4, 32, k, 4, 4).permute(0, 3, 4, 2, 1, 5).contiguous()
        self._hold(codes, int(pitch), laid.view(-1), scale.resolve_neg().contiguous(), cols)

    def _hold(self, codes, pitch, blocks, scale, cols):
        self.codes, self.pitch, self.blocks, self.scale, self.cols = codes, pitch, blocks, scale, cols
        self.index = codes.device.index
        return self

    @property
    def shape(self):
        return (self.codes.shape[0], self.cols)

    @property
    def device(self):
        return self.codes.device

    @property
    def block_scale(self):
        """The block scales as float8_e4m3fn [rows, ceil(cols / 16)]."""
        torch = _torch()
        rows, cols = self.shape
        m, k = -(-rows // 128), -(-cols // 256)
        laid = self.blocks.view(m, k, 4, 32, 4, 4).permute(0, 4, 3, 1, 2, 5).reshape(m * 128, k * 16)
        return laid[:rows, : -(-cols // BLOCK)].contiguous().view(torch.float8_e4m3fn)

    def dequantize(self):
        """The float32 matrix that the codes and scales stand for.  It has no derivative: a scale that requires one is refused."""
        refuse_grad("the scale", self.scale, "the values of 4-bit rows")
        with on_device(self.device):
            made = nat.bound_hostcall().fp4_values(self.codes, self.pitch, self.blocks, self.scale, self.cols,
                                                   raw_stream(self.index))
        if type(made) is int:
            nat.check(made, "tthrml_fp4_values")
        return made


def _readable(x):
    """A float matrix as the quantisation reads it: columns one behind the other and no negated view, or copied to be so."""
    x = x.resolve_neg()
    if x.shape[1] > 1 and x.stride(1) != 1:
        return x.contiguous()
    return x


def quantize_fp4(x) -> Fp4Rows:
    """Rows of a float32, bfloat16 or float16 matrix in 4 bits, with a scale per 16 columns and one per row.

    scale = max|x_r| / 2688, block = e4m3(max|x_b| / (6 scale)), code = e2m1(x /
    (block scale)), rounded to nearest even step by step in float32.  A row of zeros
    (or of magnitudes below 2^-100) gets scale 0, a row that holds an infinity or
    NaN gets scale NaN.  Any strides (matrices whose columns are not one behind the
    other are copied first).
    """
    torch = _torch()
    if isinstance(x, torch.Tensor) and x.is_cuda and current_device() == x.get_device():  # the plain case
        index = x.get_device()
        nat.bind_device(index)
        made = nat.bound_hostcall().quantize_fp4(x, raw_stream(index), index)
        if type(made) is int:
            nat.check(made, "tthrml_fp4_quantize")
        if made is not None:
            (rows, cols), (codes, blocks, scale) = x.shape, made
            return Fp4Rows.__new__(Fp4Rows)._hold(codes[:, : -(-cols // 2)], codes.shape[1], blocks, scale, cols)
    require_cuda("x", x)
    code = dtype_code(x.dtype)
    if code is None or x.dim() != 2:
        raise ValueError(f"x must be a float32, bfloat16 or float16 matrix, got {x.dtype} of shape {tuple(x.shape)}")
    _no_grad("x", x)
    rows, cols = x.shape
    _check_cols(cols)
    bytes_, pitch = -(-cols // 2), -(-cols // 32) * 16
    codes = torch.empty((rows, pitch), dtype=torch.uint8, device=x.device)
    blocks = torch.empty(_scale_bytes(rows, cols), dtype=torch.uint8, device=x.device)
    scale = torch.empty(rows, dtype=torch.float32, device=x.device)
    if rows:
        with on_device(x.device):
            x = _readable(x)
            nat.check(
                nat.lib().tthrml_fp4_quantize(x.data_ptr(), code, rows, cols, x.stride(0), 1, codes.data_ptr(), pitch,
                                              blocks.data_ptr(), scale.data_ptr(), raw_stream(x.device.index)),
                "tthrml_fp4_quantize",
            )
    return Fp4Rows.__new__(Fp4Rows)._hold(codes[:, :bytes_], pitch, blocks, scale, cols)


def fp4_product(x, weights: Fp4Rows, *, bias=None, out_dtype=None, out=None):
    """y = x w^T with 4-bit values: x [..., K] (float rows, quantised here, or Fp4Rows), weights [N, K].

    bias: float32 [N] added after the scaling.  out_dtype: float32, bfloat16
    or float16 (default: x's type; float32 for Fp4Rows).  out: a tensor [..., N]
    to write, its rows dense.  The sums are float32 on the tensor cores, whose additions
    cut off: sums of values of one sign are low by up to 1.4e-6 of themselves at 8192
    columns and 4.4e-5 at 2^20; values of both signs come out within 1e-7 of the norm at any
    length.  The result is the same every time.
    """
    if out is None and out_dtype is None and type(weights) is Fp4Rows:
        index = weights.index
        word = _error_addresses.get(index)
        if word is not None and current_device() == index:  # the plain case, from the second call on
            nat.bind_device(index)
            y = nat.bound_hostcall().fp4_product(x, weights.codes, weights.pitch, weights.blocks, weights.scale, weights.cols,
                                                 bias, word, raw_stream(index), index)
            if y is not None:
                if type(y) is int:
                    nat.check(y, "tthrml_fp4_linear")
                return y
    torch = _torch()
    if not isinstance(weights, Fp4Rows):
        raise TypeError(f"weights must be Fp4Rows (see quantize_fp4), got {type(weights).__name__}")
    dev, (N, K) = weights.device, weights.shape
    quantized = isinstance(x, Fp4Rows)
    rows = x.codes if quantized else x
    require_cuda("x", rows, dev)
    code = None if quantized else dtype_code(x.dtype)
    if not quantized and (code is None or x.dim() < 1):
        raise ValueError(f"x must hold float32, bfloat16 or float16 rows, got {x.dtype} of shape {tuple(x.shape)}")
    if not quantized:
        _no_grad("x", x)
    for name, q in (("x", x), ("weights", weights)):
        if isinstance(q, Fp4Rows):
            _no_grad(f"the scale of {name}", q.scale)
    lead, cols = x.shape[:-1], x.shape[-1]
    if cols != K:
        raise ValueError(f"x has rows of {cols}, the weights have {K} columns")
    if bias is not None:
        require_cuda("bias", bias, dev)
        if bias.dtype != torch.float32 or bias.shape != (N,):
            raise ValueError(f"bias must be float32 of shape ({N},), got {bias.dtype} of {tuple(bias.shape)}")
        _no_grad("bias", bias)
        bias = bias.resolve_neg().contiguous()
    if out_dtype is None:
        out_dtype = out.dtype if out is not None else (torch.float32 if quantized else x.dtype)
    out_code = dtype_code(out_dtype)
    if out_code is None:
        raise ValueError(f"out_dtype must be float32, bfloat16 or float16, got {out_dtype}")
    if out is None:
        out, out_ld = torch.empty((*lead, N), dtype=out_dtype, device=dev), N
    else:
        require_cuda("out", out, dev)
        if out.dtype != out_dtype or out.shape != (*lead, N):
            raise ValueError(f"out must be {out_dtype} of shape {(*lead, N)}, got {out.dtype} of {tuple(out.shape)}")
        refuse_written_grad("out", out)
        if out.is_neg():
            raise ValueError("out is a negated view, which the kernel cannot write")
        flat = out.view(-1, N) if N else out  # raises if the rows cannot be one matrix
        if flat.numel() and ((N > 1 and flat.stride(1) != 1) or (flat.shape[0] > 1 and flat.stride(0) < N)):
            raise ValueError("out needs dense rows that do not overlap")
        inputs = [(f"{what} of {name}", t) for name, q in (("x", x), ("the weights", weights)) if isinstance(q, Fp4Rows)
                  for what, t in (("codes", q.codes), ("block scales", q.blocks), ("scales", q.scale))]
        if not quantized:
            inputs.append(("x", x))
        if bias is not None:
            inputs.append(("bias", bias))
        refuse_overlap("out", out, inputs)
        out_ld = flat.stride(0) if N and flat.shape[0] > 1 else N
        if out.numel():
            mark_written(out)
    if not out.numel():
        return out
    lib = nat.lib()
    w_at = (weights.codes.data_ptr(), weights.pitch, weights.blocks.data_ptr(), weights.scale.data_ptr())
    with on_device(dev):
        stream, error = raw_stream(dev.index), error_word(dev).data_ptr()
        if quantized:
            nat.check(
                lib.tthrml_fp4_product(x.codes.data_ptr(), x.pitch, x.blocks.data_ptr(), x.scale.data_ptr(), *w_at, lead[0], N, K,
                                       nat.ptr(bias), out.data_ptr(), out_code, out_ld, error, stream),
                "tthrml_fp4_product",
            )
            return out
        rows = _readable(x.reshape(-1, K))
        size = lib.tthrml_fp4_linear_workspace(rows.shape[0], K, N)
        space = torch.empty(size, dtype=torch.uint8, device=dev) if size else None
        nat.check(
            lib.tthrml_fp4_linear(rows.data_ptr(), code, rows.shape[0], K, rows.stride(0), 1, nat.ptr(space), size, *w_at, N,
                                  nat.ptr(bias), out.data_ptr(), out_code, out_ld, error, stream),
            "tthrml_fp4_linear",
        )
    return out


__all__ = ["Fp4Rows", "quantize_fp4", "fp4_product"]
