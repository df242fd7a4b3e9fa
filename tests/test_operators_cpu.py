"""Operators' argument checks on the CPU: rejected calls touch neither the device nor the stand-in pointers."""

import contextlib
import ctypes
import gc
import threading

import numpy as np
import pytest
import torch

import tt_thrml_b200 as tt
from tt_thrml_b200 import _native as nat, compiler, workloads

_A, _M = 4096, 4100  # a 16-byte aligned and a misaligned stand-in address


def phases(n=1, **kw):
    rows = (nat.MomentPhase * n)()
    for r in rows:
        r.x, r.y, r.x_ld, r.y_ld, r.chains = _A, _A, 64, 64, 10
        for k, v in kw.items():
            setattr(r, k, v)
    return rows


def tensors(**kw):
    rows = (nat.AdamWTensor * 1)()
    rows[0].param, rows[0].grad, rows[0].n, rows[0].state = _A, _A, 5, 0
    for k, v in kw.items():
        setattr(rows[0], k, v)
    return rows


def quantize(x=_A, dtype=0, rows=2, cols=40, rs=40, cs=1, values=_A, pitch=48, scale=_A):
    return x, dtype, rows, cols, rs, cs, values, pitch, scale, None


def product(x=_A, xp=48, w=_A, wp=48, ws=_A, rows=20, units=8, cols=40, out=_A, dt=0, ld=8, err=_A):
    return x, xp, None, w, wp, ws, rows, units, cols, None, out, dt, ld, err, None


def few(x=_A, xd=1, ld=40, w=_A, wp=48, rows=2, units=8, cols=40, out=_A, od=0, old=8):
    return x, xd, ld, None, w, wp, _A, rows, units, cols, None, out, od, old, None


def field(src=_A, sp=64, w=_A, wp=64, ws=_A, c=128, n=256, k=64, bias=None, family=0, out=_A, offset=0, err=_A):
    return src, sp, None, w, wp, ws, c, n, k, bias, family, 1.0, out, 0, offset, None, 0, 0, 0, None, err, None


def moments(ph, n=1, dt=1, m=8, k=8, out=_A, ld=8, err=_A):
    return ph, n, dt, m, k, out, ld, None, None, 0, err, None


def linear(x=_A, dt=1, rows=20, cols=40, rs=40, cs=1, ws=None, size=0, w=_A, wp=48, scale=_A, units=8, out=_A, od=1, ld=8, err=_A):
    return x, dt, rows, cols, rs, cs, ws, size, w, wp, scale, units, None, out, od, ld, err, None


def pack(**kw):
    rows = (nat.PackMatrix * 1)()
    r = rows[0]
    r.src, r.dst, r.rows, r.cols, r.row_stride, r.col_stride, r.pitch = _A, _A, 3, 5, 5, 1, 8
    for k, v in kw.items():
        setattr(r, k, v)
    return rows


def adamw(t, n=1, bits=32, m=_A, v=_A, ms=None, vs=None, ctl=_A, b1=0.9, b2=0.99, eps=1e-8, wd=0.0):
    return t, n, bits, m, v, ms, vs, ctl, b1, b2, eps, wd, 0, None


BAD = [
    ("tthrml_quantize_rows", quantize(x=None), b"NULL"),
    ("tthrml_quantize_rows", quantize(cols=0), b"out of range"),
    ("tthrml_quantize_rows", quantize(cs=0), b"out of range"),
    ("tthrml_quantize_rows", quantize(pitch=40), b"multiple of 16"),
    ("tthrml_quantize_rows", quantize(pitch=32), b"multiple of 16"),
    ("tthrml_quantize_rows", quantize(values=_M), b"16-byte aligned"),
    ("tthrml_quantize_rows", quantize(dtype=3), b"input type"),
    ("tthrml_widen_i8", (_A, 5, _M, None), b"16-byte aligned"),
    ("tthrml_widen_i8", (None, 5, _A, None), b"must be given"),
    ("tthrml_int8_product", product(err=None), b"NULL"),
    ("tthrml_int8_product", product(cols=131072, xp=131072, wp=131072), b"out of range"),
    ("tthrml_int8_product", product(rows=-1), b"out of range"),
    ("tthrml_int8_product", product(dt=3), b"output type"),
    ("tthrml_int8_product", product(dt=9), b"output type"),
    ("tthrml_int8_product", product(x=_M), b"16-byte aligned"),
    ("tthrml_int8_product", product(wp=40), b"16-byte aligned"),
    ("tthrml_int8_product", product(xp=32), b"16-byte aligned"),
    ("tthrml_int8_product", product(ld=7), b"must not overlap"),
    ("tthrml_int8_product_few", few(w=None), b"NULL"),
    ("tthrml_int8_product_few", few(rows=3), b"1 or 2 rows"),
    ("tthrml_int8_product_few", few(rows=2, cols=82000, ld=82000, wp=82000), b"shared memory"),
    ("tthrml_int8_product_few", few(xd=7), b"unknown element type"),
    ("tthrml_int8_product_few", few(od=3), b"unknown element type"),
    ("tthrml_int8_product_few", few(ld=39), b"must not overlap"),
    ("tthrml_int8_product_few", few(w=_M), b"16-byte aligned"),
    ("tthrml_int8_field_sample", field(out=None), b"NULL"),
    ("tthrml_int8_field_sample", field(n=40), b"multiple of 32"),
    ("tthrml_int8_field_sample", field(k=131072, sp=131072, wp=131072), b"at most"),
    ("tthrml_int8_field_sample", field(family=1), b"spin or gaussian"),
    ("tthrml_int8_field_sample", field(offset=2), b"chain_offset"),
    ("tthrml_int8_field_sample", field(bias=_M), b"16-byte aligned"),
    ("tthrml_int8_field_sample", field(sp=60), b"pitches"),
    ("tthrml_pair_moments", moments(None), b"NULL"),
    ("tthrml_pair_moments", moments(phases(7), n=7), b"1 to 6 phases"),
    ("tthrml_pair_moments", moments(phases(), dt=0), b"bfloat16 or float16"),
    ("tthrml_pair_moments", moments(phases(), m=0), b"out of range"),
    ("tthrml_pair_moments", moments(phases(), ld=7), b"out of range"),
    ("tthrml_pair_moments", moments(phases(x=_M)), b"16-byte aligned"),
    ("tthrml_pair_moments", moments(phases(y_ld=60)), b"16-byte aligned"),
    ("tthrml_pair_moments", moments(phases(x_ld=8), m=9), b"16-byte aligned"),
    ("tthrml_pair_moments", moments(phases(chains=-1)), b"16-byte aligned"),
    ("tthrml_int8_linear", linear(), b"workspace"),
    ("tthrml_int8_linear", linear(ws=_A, size=979), b"needs a 16-byte aligned workspace of 1040 bytes"),
    ("tthrml_int8_linear", linear(ws=_M, size=4096), b"workspace"),
    ("tthrml_int8_linear", linear(rows=1, cs=2), b"workspace"),
    ("tthrml_int8_linear", linear(rows=2, rs=39), b"workspace"),
    ("tthrml_int8_linear", linear(cols=0), b"out of range"),
    ("tthrml_int8_linear", linear(rows=2, w=None), b"NULL"),
    ("tthrml_int8_linear", linear(rows=1, dt=9), b"unknown element type"),
    ("tthrml_pack_rows", (None, 1, None), b"matrices"),
    ("tthrml_pack_rows", (pack(), 13, None), b"0 to 12 matrices"),
    ("tthrml_pack_rows", (pack(pitch=4), 1, None), b"matrix 0"),
    ("tthrml_pack_rows", (pack(pitch=12), 1, None), b"matrix 0"),
    ("tthrml_pack_rows", (pack(dst=_M), 1, None), b"matrix 0"),
    ("tthrml_pack_rows", (pack(src=_A + 1), 1, None), b"matrix 0"),
    ("tthrml_pair_moments_packed", (pack(rows=-1), 1, *moments(phases())), b"matrix 0"),
    ("tthrml_adamw_step", adamw(None), b"NULL"),
    ("tthrml_adamw_step", adamw(tensors(), bits=8), b"NULL"),
    ("tthrml_adamw_step", adamw(tensors(), bits=16), b"8 or 32"),
    ("tthrml_adamw_step", adamw(tensors(), b1=1.0), b"betas"),
    ("tthrml_adamw_step", adamw(tensors(), eps=0.0), b"eps"),
    ("tthrml_adamw_step", adamw(tensors(), b2=float("nan")), b"betas"),
    ("tthrml_adamw_step", adamw(tensors(), m=_M), b"16-byte aligned"),
    ("tthrml_adamw_step", adamw(tensors(n=0)), b"tensor 0"),
    ("tthrml_adamw_step", adamw(tensors(state=128)), b"tensor 0"),
    ("tthrml_adamw_step", adamw(tensors(param_dtype=3)), b"tensor 0"),
    ("tthrml_adamw_step", adamw(tensors(grad=_A + 2)), b"tensor 0"),
    ("tthrml_adamw_values", (_A, _A, _A, _A, 100, _A, _A, None), b"multiple of 256"),
    ("tthrml_adamw_values", (None, _A, _A, _A, 256, _A, _A, None), b"NULL"),
]


@pytest.mark.parametrize("name,args,message", BAD, ids=[f"{c[0]}-{i}" for i, c in enumerate(BAD)])
def test_bad_arguments_are_rejected_before_any_cuda_call(name, args, message):
    lib = nat.lib()
    assert getattr(lib, name)(*args) == -1
    assert message in lib.tthrml_last_error(), lib.tthrml_last_error()


@pytest.mark.parametrize("name,args", [
    ("tthrml_quantize_rows", quantize(rows=0, x=None)),
    ("tthrml_int8_product", product(rows=0, x=None)),
    ("tthrml_int8_product", product(units=0, w=None)),
    ("tthrml_int8_product_few", few(rows=0, x=None)),
    ("tthrml_int8_linear", linear(rows=0, x=None)),
    ("tthrml_int8_linear", linear(units=0, w=None)),
    ("tthrml_pack_rows", (None, 0, None)),
    ("tthrml_pack_rows", (pack(rows=0, src=None), 1, None)),
    ("tthrml_adamw_step", adamw(None, n=0)),
    ("tthrml_adamw_values", (None, None, None, None, 0, None, None, None)),
])
def test_empty_calls_do_nothing(name, args):
    assert getattr(nat.lib(), name)(*args) == 0


def test_structures_have_the_header_layout():
    assert ctypes.sizeof(nat.AdamWTensor) == 40 and ctypes.sizeof(nat.MomentPhase) == 56
    assert ctypes.sizeof(nat.PackMatrix) == 56 and ctypes.sizeof(nat.AdamWCall) == 104


def test_workspace_of_the_linear_entry():
    lib = nat.lib()
    assert lib.tthrml_int8_linear_workspace(1, 163840) == 0 and lib.tthrml_int8_linear_workspace(2, 81920) == 0
    assert lib.tthrml_int8_linear_workspace(2, 81921) == 2 * 81936 + 16
    assert lib.tthrml_int8_linear_workspace(20, 40) == 20 * 48 + 80


def test_host_module_leaves_other_cases_to_python():
    host, x = nat.hostcall(), torch.ones((2, 4))
    assert host.int8_product(x, x, x[0], 16, None, 0, 0, 0, 0) is None
    assert host.int8_product("x", x, x[0], 16, None, 0, 0, 0, 0) is None
    assert host.pair_moments([x], [x], [1.0], False, 0, 0, 0, 0, 0) is None
    assert host.pair_moments([x], [], [1.0], False, 0, 0, 0, 0, 0) is None
    call = nat.AdamWCall()
    assert host.adamw_step([x], [x], ctypes.addressof(call), 0, 0, 0) == 0  # the first pair is not on the device
    assert host.adamw_step([x], [None], ctypes.addressof(call), 0, 0, 0) == 0
    for bad in ((), ([x], [x, x], 0, 0, 0, 0), ((x,), [x], 0, 0, 0, 0)):
        with pytest.raises(TypeError):
            host.adamw_step(*bad)
    for bad in ((0,), (0, 1, 256, 0, 0), (0, "codes", 256, 0, 0)):
        with pytest.raises(TypeError):
            host.adamw_values(*bad)
    version = x._version
    host.bump_versions([x, 3])
    assert x._version == version + 1
    with pytest.raises(TypeError):
        host.bump_versions(x)


def test_cpu_tensors_are_refused():
    x = torch.ones((2, 3))
    for call in (lambda: tt.quantize_rows(x), lambda: tt.QuantizedRows(x.to(torch.int8)), lambda: tt.AdamW([x]),
                 lambda: tt.pair_moments(x.bfloat16(), x.bfloat16())):
        with pytest.raises(ValueError, match="CUDA"):
            call()
    with pytest.raises(TypeError):
        tt.int8_product(x, x)
    with pytest.raises(ValueError):
        tt.AdamW([])


def test_host_quantisation_and_the_int8_plan():
    r = np.random.default_rng(0)
    w = r.standard_normal((5, 37)).astype(np.float32)
    w[2] = 0.0
    q, s = compiler.quantize_rows_host(w)
    assert q.shape == (5, 48) and not q[:, 37:].any() and not q[2].any() and s[2] == 0.0
    assert np.abs(q).max(1)[[0, 1, 3, 4]].tolist() == [127] * 4
    # half a step of the row's scale, and float32 roundings
    assert (np.abs(q[:, :37] * s[:, None].astype(np.float64) - w) <= s[:, None] * (0.5 + 1e-4)).all()
    w[1, 1] = np.inf
    with pytest.raises(ValueError):
        compiler.quantize_rows_host(w)
    program = workloads.gaussian_bernoulli_rbm(256, 512, seed=1)
    plans = compiler._plan_dense(program, torch.device("cpu"), "int8")
    assert [p.weights_nk.dtype for p in plans] == [torch.int8] * 2 and all(p.w_scale is not None for p in plans)
    with pytest.raises(ValueError):
        tt.make_cuda_config(dense_precision="int4")
    a, b = tt.make_cuda_config(dense_precision="int8"), tt.make_cuda_config(dense_precision="bf16")
    assert a.resolved_dense_precision == "int8" and a.plan_key() != b.plan_key()


def test_an_error_on_another_device_leaves_no_binding(monkeypatch):
    """The library's device is looked up again after a call on a device that is not current, also one that raises."""
    import contextlib
    import types

    from tt_thrml_b200 import quantized

    bound = []
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
    monkeypatch.setattr(torch.cuda, "device", lambda index: contextlib.nullcontext())
    monkeypatch.setattr(nat, "lib", lambda: types.SimpleNamespace(tthrml_set_device=lambda i: bound.append(i) or nat.OK))
    monkeypatch.setattr(nat, "_bound", types.SimpleNamespace())
    with pytest.raises(RuntimeError, match="inside"):
        with quantized.on_device(torch.device("cuda", 1)):
            assert nat._bound.device == 1
            raise RuntimeError("inside")
    assert nat._bound.device is None
    nat.bind_device(0)
    assert bound == [1, 0]


def test_outputs_that_share_memory_are_refused():
    from tt_thrml_b200.quantized import refuse_shared_outputs

    buffer = torch.zeros(100)
    out, x_sum, y_sum = buffer[:25].view(5, 5), buffer[25:30], buffer[30:35]
    refuse_shared_outputs([("out", out), ("x_sum", x_sum), ("y_sum", y_sum)])
    refuse_shared_outputs([("out", out[:0]), ("x_sum", buffer[:0])])
    for outs in ([out, x_sum, x_sum], [out, out[2], y_sum], [out, buffer[24:29], y_sum], [out, x_sum, buffer[29:34]]):
        with pytest.raises(ValueError, match="share memory"):
            refuse_shared_outputs(list(zip(("out", "x_sum", "y_sum"), outs)))


def test_an_expired_wait_is_reported_once(monkeypatch):
    from tt_thrml_b200 import quantized

    words = {0: torch.tensor([3], dtype=torch.int32), 1: torch.tensor([1], dtype=torch.int32), 2: torch.zeros(1, dtype=torch.int32)}
    monkeypatch.setattr(quantized, "_error_words", words)
    monkeypatch.setattr(torch.cuda, "synchronize", lambda index=None: None)
    tt.check_operator_errors("cuda:2")
    with pytest.raises(RuntimeError, match=r"code 1, device 1"):
        tt.check_operator_errors(torch.device("cuda", 1))
    tt.check_operator_errors("cuda:1")
    words[1].fill_(2)
    with pytest.raises(RuntimeError, match=r"code 3, device 0.*code 2, device 1"):
        tt.check_operator_errors()
    tt.check_operator_errors()
    assert not any(w.item() for w in words.values())


@pytest.mark.parametrize("ran", [True, False])
def test_captures_in_two_threads_pause_the_collector_together(monkeypatch, ran):
    monkeypatch.setattr(torch.cuda, "graph", lambda graph, stream=None: contextlib.nullcontext())
    started, finish, seen = threading.Event(), threading.Event(), []

    def other():
        with nat.capturing(None):
            started.set()
            finish.wait(10)
            seen.append(gc.isenabled())

    was = gc.isenabled()
    (gc.enable if ran else gc.disable)()
    try:
        thread = threading.Thread(target=other)
        with nat.capturing(None):
            thread.start()
            assert started.wait(10) and not gc.isenabled()
        assert not gc.isenabled()  # the other thread still captures
        finish.set()
        thread.join(10)
        assert seen == [False] and gc.isenabled() is ran
        with pytest.raises(RuntimeError, match="inside"):
            with nat.capturing(None):
                raise RuntimeError("inside")
        assert gc.isenabled() is ran
    finally:
        finish.set()
        (gc.enable if was else gc.disable)()


def test_the_host_module_is_made_again_for_another_torch(monkeypatch, tmp_path):
    from tt_thrml_b200 import build

    made = []

    def compiler(cmd, check):
        assert check
        made.append(cmd)
        with open(cmd[cmd.index("-o") + 1], "w") as f:
            f.write("module")

    monkeypatch.setattr(build.subprocess, "run", compiler)
    monkeypatch.setattr(build, "BUILD_DIR", tmp_path / "objects")
    monkeypatch.setattr(build, "HOSTCALL_PATH", tmp_path / "_hostcall.so")
    for count in (1, 1):
        assert build.build_hostcall() == tmp_path / "_hostcall.so" and len(made) == count
    with monkeypatch.context() as other:
        other.setattr(torch, "__version__", torch.__version__ + ".other")
        for count in (2, 2):
            build.build_hostcall()
            assert len(made) == count
    build.build_hostcall()
    with monkeypatch.context() as other:
        other.setattr(build.sys, "version", "another Python")
        build.build_hostcall()
    assert len(made) == 4
    build.build_hostcall(force=True)
    assert len(made) == 5


def views(base, seed):
    """A view of a few rows and columns, of any strides, into a buffer of 600 elements."""
    r = np.random.default_rng(seed)
    pitch = int(r.choice([7, 12, 20]))
    m = base[: 600 // pitch * pitch].view(-1, pitch)
    r0, c0 = int(r.integers(0, 20)), int(r.integers(0, pitch))
    v = m[r0 : r0 + int(r.integers(1, 9)), c0 : c0 + int(r.integers(1, 9))]
    kind = r.integers(0, 6)
    if kind == 0:
        return v[::2]
    if kind == 1:
        return v.t()
    if kind == 2:
        return v[0]
    if kind == 3:
        return v[:, ::2]
    if kind == 4:
        return v[: v.shape[0] // 2 * 2].unflatten(0, (-1, 2)) if v.shape[0] > 1 else v
    return v


def test_views_that_share_memory():
    """Against the elements themselves: nothing shared passes, and ranges of columns of one matrix do not collide."""
    from tt_thrml_b200.quantized import share_memory

    kept, base = 0, torch.arange(600)  # an element's value is its place
    for i in range(6000):
        a, b = views(base, 2 * i), views(base, 2 * i + 1)
        shared = bool(set(a.flatten().tolist()) & set(b.flatten().tolist()))
        assert not shared or (share_memory(a, b) and share_memory(b, a)), (i, a.shape, a.stride(), b.shape, b.stride())
        kept += not shared and not share_memory(a, b)
    assert kept > 2000
    both = torch.zeros(6, 20)
    x, out = both[:, :8], both[:, 8:]
    assert not share_memory(out, x) and not share_memory(x, out)
    assert share_memory(both[:, :9], out) and share_memory(out, both[:, :9]) and share_memory(both[1:3, 19:], out)
    assert not share_memory(both[2, :8], out) and not share_memory(out, both[5:, :8])
    assert share_memory(out, both[2, 7:9]) and not share_memory(both[:0], both)
    assert not share_memory(both.view(2, 3, 20)[:, :, :8], both.view(2, 3, 20)[..., 8:])
