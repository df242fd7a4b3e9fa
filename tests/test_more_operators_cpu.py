"""The readout's operators on the CPU: rejected calls touch neither the device nor the stand-in pointers."""

import ctypes

import pytest
import torch

import tt_thrml_b200 as tt
from tt_thrml_b200 import _native as nat

_A, _M = 4096, 4104  # a 16-byte aligned and a misaligned stand-in address


def xent(**kw):
    p = nat.Xent()
    p.x = p.w = p.targets = _A
    p.x_ld = p.w_ld = 64
    p.rows, p.categories, p.cols, p.ignored, p.dtype, p.wide_targets = 10, 20, 60, -100, nat.DT_BF16, 1
    for k, v in kw.items():
        setattr(p, k, v)
    return p


def forward(z=_A, row_loss=_A, loss=_A, inv=_A, reduction=1, ws=_A, size=1 << 20, err=_A, **kw):
    return xent(**kw), z, row_loss, loss, inv, reduction, ws, size, err, None


def backward(z=_A, grad=_A, per_row=0, inv=_A, dx=_A, dx_ld=60, dw=_A, dw_ld=60, dtype=1, db=_A, ws=_A, size=1 << 20, err=_A, **kw):
    return xent(**kw), z, grad, per_row, inv, dx, dx_ld, dw, dw_ld, dtype, db, ws, size, err, None


def dropout(x=_A, dtype=0, n=10, cut=5, seed=1, step=0, at=None, wide=0, used=None, y=_A):
    return x, dtype, n, cut, seed, step, at, wide, used, y, None


def quantize(x=_A, dtype=0, rows=2, cols=40, rs=40, cs=1, codes=_A, pitch=32, blocks=_A, scale=_A):
    return x, dtype, rows, cols, rs, cs, codes, pitch, blocks, scale, None


def values(codes=_A, pitch=32, blocks=_A, scale=_A, rows=2, cols=40, out=_A):
    return codes, pitch, blocks, scale, rows, cols, out, None


def product(xc=_A, xp=32, xb=_A, xs=_A, wc=_A, wp=32, wb=_A, ws=_A, rows=20, units=8, cols=40, out=_A, dt=0, ld=8, err=_A):
    return xc, xp, xb, xs, wc, wp, wb, ws, rows, units, cols, None, out, dt, ld, err, None


def linear(x=_A, dt=1, rows=20, cols=40, rs=40, cs=1, ws=None, size=0, wc=_A, wp=32, units=8, out=_A, od=1, ld=8, err=_A):
    return x, dt, rows, cols, rs, cs, ws, size, wc, wp, _A, _A, units, None, out, od, ld, err, None


def few(x=_A, dt=1, ld=40, wc=_A, wp=32, rows=2, units=8, cols=40, out=_A, od=0, old=8, err=_A):
    return x, dt, ld, wc, wp, _A, _A, rows, units, cols, None, out, od, old, err, None


BAD = [
    ("tthrml_xent_forward", forward(x=None), b"NULL"),
    ("tthrml_xent_forward", forward(targets=None), b"NULL"),
    ("tthrml_xent_forward", forward(z=None), b"NULL"),
    ("tthrml_xent_forward", forward(loss=None), b"NULL"),
    ("tthrml_xent_forward", forward(reduction=3), b"reduction 3"),
    ("tthrml_xent_forward", forward(dtype=nat.DT_F32), b"bfloat16 or float16"),
    ("tthrml_xent_forward", forward(rows=0), b"out of range"),
    ("tthrml_xent_forward", forward(rows=nat.XENT_MAX_ROWS + 1), b"out of range"),
    ("tthrml_xent_forward", forward(categories=0), b"out of range"),
    ("tthrml_xent_forward", forward(cols=nat.XENT_MAX_COLS + 1), b"out of range"),
    ("tthrml_xent_forward", forward(x=_M), b"16-byte aligned"),
    ("tthrml_xent_forward", forward(w_ld=60), b"multiples of 8"),
    ("tthrml_xent_forward", forward(x_ld=56), b"not below the columns"),
    ("tthrml_xent_forward", forward(targets=_A + 4), b"aligned"),
    ("tthrml_xent_backward", backward(w=None), b"NULL"),
    ("tthrml_xent_backward", backward(grad=None), b"NULL"),
    ("tthrml_xent_backward", backward(dx_ld=59), b"rows overlap"),
    ("tthrml_xent_backward", backward(dw_ld=59), b"rows overlap"),
    ("tthrml_xent_backward", backward(dtype=nat.DT_I8), b"code 3"),
    ("tthrml_dropout", dropout(x=None), b"NULL"),
    ("tthrml_dropout", dropout(dtype=3), b"code 3"),
    ("tthrml_dropout", dropout(cut=-1), b"out of range"),
    ("tthrml_dropout", dropout(cut=65537), b"out of range"),
    ("tthrml_dropout", dropout(n=-1), b"out of range"),
    ("tthrml_dropout", dropout(x=4098), b"alignment"),
    ("tthrml_dropout", dropout(at=4100, wide=1), b"alignment"),
    ("tthrml_fp4_quantize", quantize(x=None), b"NULL"),
    ("tthrml_fp4_quantize", quantize(scale=None), b"NULL"),
    ("tthrml_fp4_quantize", quantize(cols=0), b"out of range"),
    ("tthrml_fp4_quantize", quantize(cols=nat.FP4_MAX_COLS + 1, pitch=1 << 20), b"out of range"),
    ("tthrml_fp4_quantize", quantize(pitch=16), b"holds the columns"),
    ("tthrml_fp4_quantize", quantize(pitch=24), b"multiple of 16"),
    ("tthrml_fp4_quantize", quantize(blocks=_M), b"16-byte aligned"),
    ("tthrml_fp4_quantize", quantize(cs=0), b"strides"),
    ("tthrml_fp4_quantize", quantize(dtype=3), b"input type"),
    ("tthrml_fp4_values", values(out=_M), b"16-byte aligned"),
    ("tthrml_fp4_values", values(codes=None), b"NULL"),
    ("tthrml_fp4_product", product(xb=None), b"NULL"),
    ("tthrml_fp4_product", product(cols=0), b"out of range"),
    ("tthrml_fp4_product", product(rows=-1), b"out of range"),
    ("tthrml_fp4_product", product(rows=1 << 27, units=1 << 27, ld=1 << 27), b"out of range"),
    ("tthrml_fp4_product", product(dt=3), b"output type"),
    ("tthrml_fp4_product", product(xp=16), b"hold the columns"),
    ("tthrml_fp4_product", product(wc=_M), b"16-byte aligned"),
    ("tthrml_fp4_product", product(ld=7), b"overlap"),
    ("tthrml_fp4_linear", linear(), b"workspace"),
    ("tthrml_fp4_linear", linear(ws=_M, size=1 << 20), b"16-byte aligned workspace"),
    ("tthrml_fp4_linear", linear(cols=0), b"out of range"),
    ("tthrml_fp4_linear", linear(rows=2, cs=2), b"dense columns"),
    ("tthrml_fp4_product_few", few(x=None), b"NULL"),
    ("tthrml_fp4_product_few", few(err=None), b"NULL"),
    ("tthrml_fp4_product_few", few(rows=5), b"1 to 4 rows"),
    ("tthrml_fp4_product_few", few(od=3), b"output type"),
    ("tthrml_fp4_product_few", few(wp=24), b"multiple of 16"),
    ("tthrml_fp4_product_few", few(old=7), b"overlap"),
]


@pytest.mark.parametrize("name,args,message", BAD, ids=[f"{n}-{i}" for i, (n, _, _) in enumerate(BAD)])
def test_bad_arguments_are_refused(name, args, message):
    fn = getattr(nat.lib(), name)
    assert fn(*[ctypes.byref(a) if isinstance(a, nat.Xent) else a for a in args]) == -1
    assert message in nat.lib().tthrml_last_error(), nat.lib().tthrml_last_error()


def test_nothing_to_do_is_no_error():
    lib = nat.lib()
    assert lib.tthrml_dropout(*dropout(n=0, x=None, y=None)) == 0
    assert lib.tthrml_fp4_quantize(*quantize(rows=0, x=None)) == 0
    assert lib.tthrml_fp4_values(*values(rows=0, codes=None)) == 0
    assert lib.tthrml_fp4_product(*product(rows=0, xc=None)) == 0
    assert lib.tthrml_fp4_product(*product(units=0, xc=None)) == 0
    assert lib.tthrml_fp4_linear(*linear(rows=0, x=None)) == 0
    assert lib.tthrml_xent_backward(*backward(dx=None, dw=None, db=None)) == 0


def test_sizes_of_4_bit_rows():
    lib = nat.lib()
    assert lib.tthrml_fp4_scale_bytes(1, 1) == lib.tthrml_fp4_scale_bytes(128, 256) == 2048
    assert lib.tthrml_fp4_scale_bytes(129, 257) == 4 * 2048
    assert lib.tthrml_fp4_few_rows(4, 32768, 18944) == 1
    for sizes in ((5, 64, 64), (0, 64, 64), (1, 32769, 64), (1, 64, 18945)):
        assert lib.tthrml_fp4_few_rows(*sizes) == 0
    assert lib.tthrml_fp4_linear_workspace(4, 100, 100) == 0
    assert lib.tthrml_fp4_linear_workspace(5, 100, 100) == 5 * 64 + 2048 + 32


def test_tensors_of_the_host_are_refused():
    x, y = torch.ones(4, 8, dtype=torch.bfloat16), torch.zeros(4, dtype=torch.int64)
    for call in (lambda: tt.softmax_cross_entropy(x, x, y), lambda: tt.dropout(x, 0.5, seed=1), lambda: tt.quantize_fp4(x),
                 lambda: tt.Fp4Rows(torch.zeros(4, 4, dtype=torch.uint8), torch.zeros(4, 1, dtype=torch.float8_e4m3fn),
                                    torch.ones(4))):
        with pytest.raises(ValueError, match="there is no CPU path"):
            call()
    for call in (lambda: tt.softmax_cross_entropy([1.0], x, y), lambda: tt.dropout(1.0, 0.5, seed=1), lambda: tt.quantize_fp4(None)):
        with pytest.raises(TypeError, match="torch tensor"):
            call()
    with pytest.raises(TypeError, match="must be Fp4Rows"):
        tt.fp4_product(x, x)


def test_the_host_module_checks_its_arguments():
    host = nat.bound_hostcall()
    for name in ("softmax_cross_entropy", "softmax_cross_entropy_gradients", "dropout", "fp4_values", "bind_library"):
        with pytest.raises(TypeError, match=name):
            getattr(host, name)(1)
    assert host.quantize_fp4(1) is None and host.fp4_product(1) is None
    x = torch.ones(4, 8)
    assert host.quantize_fp4(x, 0, 0) is None  # not on the device
