"""8-bit integer products on the GPU against a plain implementation in 64 bits."""

import numpy as np
import pytest
import torch

from tt_thrml_b200 import _native as nat

pytestmark = pytest.mark.gpu

DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
F32_EPS = 2.0**-24  # half a step of float32, relative


@pytest.fixture(scope="module")
def tt():
    import tt_thrml_b200

    return tt_thrml_b200


def plain_quantize(x):
    """(q, scale) of the rows of a CPU tensor by the formula, in float32 (numpy float32 operations are IEEE)."""
    f = x.float().numpy()
    top = np.abs(f).max(1)
    live = top >= np.float32(2.0**-120)
    inv = np.zeros_like(top)
    inv[live] = np.float32(127.0) / top[live]
    q = np.clip(np.rint(f * inv[:, None]), -127, 127).astype(np.int64)
    return q, np.where(live, top * np.float32(1.0 / 127.0), np.float32(0.0))


def rand(shape, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(shape, generator=g).to(dtype)


def check_product(y, q, sx, w, sw, bias, dtype):
    """|y - exact| within the roundings of the formula: the conversion of the sum, the product of the scales and the
    scaling (three of float32, relative to the product), the bias addition (one, relative to the result) and the
    last one to the output type."""
    prod = (q.astype(np.float64) @ w.astype(np.float64).T) * np.outer(sx.astype(np.float64), sw.astype(np.float64))
    exact = prod if bias is None else prod + bias.astype(np.float64)
    half = torch.finfo(dtype).eps / 2
    tiny = float(torch.finfo(dtype).smallest_normal) * torch.finfo(dtype).eps  # one step of a subnormal output
    tol32 = 3.01 * F32_EPS * np.abs(prod) + F32_EPS * np.abs(exact)
    tol = tol32 + (half * (np.abs(exact) + tol32) if dtype != torch.float32 else 0.0) + tiny
    got = y.double().cpu().numpy()
    assert got.shape == exact.shape
    bad = np.abs(got - exact) > tol
    assert not bad.any(), (int(bad.sum()), float(np.abs(got - exact).max()))


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("rows,cols", [(1, 1), (3, 15), (8, 16), (5, 17), (33, 1000), (7, 1024), (9, 1025), (2, 4103),
                                       (4, 8192), (1, 40000)])
def test_quantize_rows_matches_the_formula(tt, rows, cols, dtype):
    x = rand((rows, cols), DTYPES[dtype], rows * 7 + cols)
    r = tt.quantize_rows(x.cuda())
    q, s = plain_quantize(x)
    assert np.array_equal(r.values.cpu().numpy(), q) and np.array_equal(r.scale.cpu().numpy(), s)
    assert r.pitch % 16 == 0 and r.shape == (rows, cols)


@pytest.mark.parametrize("dtype", list(DTYPES))
def test_quantize_rows_strides(tt, dtype):
    t = DTYPES[dtype]
    base = rand((70, 301), t, 3)
    d = base.cuda()
    for shape in ((5000, 100), (4096, 70), (17, 40), (2000, 33)):  # transposed: long rows, an odd number of them
        wide = rand(shape, t, shape[0])
        r = tt.quantize_rows(wide.cuda().t())
        q, s = plain_quantize(wide.t())
        assert np.array_equal(r.values.cpu().numpy(), q) and np.array_equal(r.scale.cpu().numpy(), s)
    cases = [(base.t(), d.t()), (base[:, ::3], d[:, ::3]), (base[1::2, 5:], d[1::2, 5:]), (base[:, 1:130], d[:, 1:130]),
             (base[:1].expand(9, 301), d[:1].expand(9, 301)), (base[:, :1].expand(70, 40), d[:, :1].expand(70, 40)),
             (base.t()[:, 3:4], d.t()[:, 3:4])]
    for cpu, gpu in cases:
        assert gpu.stride() == cpu.stride()
        r = tt.quantize_rows(gpu)
        q, s = plain_quantize(cpu)
        assert np.array_equal(r.values.cpu().numpy(), q) and np.array_equal(r.scale.cpu().numpy(), s)


@pytest.mark.parametrize("cols", [64, 1500, 9000])
def test_quantize_rows_special_values(tt, cols):
    x = rand((8, cols), torch.float32, 5)
    x[0] = 0.0
    x[1, cols // 2] = float("inf")
    x[2, cols - 1] = float("nan")
    x[3] = x[3] * 2.0**-130
    x[4] = x[4] * 1e30
    x[5, 0] = -float("inf")
    x[6] = 2.0**-119
    r = tt.quantize_rows(x.cuda())
    v, s = r.values.cpu().numpy(), r.scale.cpu().numpy()
    for row in (0, 3):
        assert s[row] == 0.0 and not v[row].any()
    for row in (1, 2, 5):
        assert np.isnan(s[row])
    q, ps = plain_quantize(x[[4, 6, 7]])
    assert np.array_equal(v[[4, 6, 7]], q) and np.array_equal(s[[4, 6, 7]], ps)
    # a row that is not finite makes its own products NaN and no others
    w = tt.quantize_rows(rand((20, cols), torch.float32, 6).cuda())
    y = tt.int8_product(x.cuda(), w)
    assert torch.isnan(y[[1, 2, 5]]).all() and torch.isfinite(y[[0, 3, 4, 6, 7]]).all()
    for r in range(8):  # the form for single rows
        one = tt.int8_product(x[r : r + 1].cuda(), w)
        assert torch.equal(torch.isnan(one[0]), torch.isnan(y[r])) and torch.equal(one[0].nan_to_num(), y[r].nan_to_num())


SHAPES = [(1, 1, 1), (1, 1, 16), (1, 130, 4096), (2, 17, 31), (3, 64, 2048), (4, 255, 5000), (5, 33, 48), (8, 129, 1023),
          (8, 40, 20480), (2, 5000, 600), (1, 3001, 12345), (2, 20, 81920), (2, 21, 81921), (9, 1, 1), (9, 130, 127), (16, 64, 128), (17, 65, 129), (37, 203, 501), (64, 128, 256),
          (100, 300, 1000), (128, 256, 512), (129, 257, 640), (300, 70, 3000), (513, 515, 259), (260, 1030, 130)]


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("rows,units,cols", SHAPES)
def test_product_matches_the_64_bit_sum(tt, rows, units, cols, dtype):
    t = DTYPES[dtype]
    x, w = rand((rows, cols), t, rows + cols), rand((units, cols), torch.float32, units)
    bias = rand((units,), torch.float32, 9) if units % 2 else None
    wq, sw = plain_quantize(w)
    q, sx = plain_quantize(x)
    r = tt.quantize_rows(w.cuda())
    y = tt.int8_product(x.cuda(), r, bias=None if bias is None else bias.cuda())
    assert y.dtype == t
    check_product(y, q, sx, wq, sw, None if bias is None else bias.numpy(), t)
    tt.check_operator_errors()


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("rows,units,cols", [(140, 8190, 700), (777, 3001, 1000), (300, 1501, 5001), (200, 3001, 6000),
                                             (257, 4500, 3333), (520, 3001, 2500), (1000, 4001, 2100),
                                             (1000, 4008, 2100)])
def test_products_of_some_hundred_rows(tt, rows, units, cols, dtype):
    """Tiles of 256 rows, whole and cut off, the columns in one share or several: exact sums on every path, so the result of
    128 rows at a time (tiles of 128) is the same to the bit."""
    t = DTYPES[dtype]
    x, w = rand((rows, cols), t, rows + cols), rand((units, cols), torch.float32, units)
    bias = rand((units,), torch.float32, 9)
    wq, sw = plain_quantize(w)
    q, sx = plain_quantize(x)
    r = tt.quantize_rows(w.cuda())
    d, b = x.cuda(), bias.cuda()
    y = tt.int8_product(d, r, bias=b)
    check_product(y, q, sx, wq, sw, bias.numpy(), t)
    parts = torch.cat([tt.int8_product(d[m : m + 128], r, bias=b) for m in range(0, rows, 128)])
    assert torch.equal(y, parts)
    assert torch.equal(tt.int8_product(tt.quantize_rows(d), r, bias=b, out_dtype=t), y)
    tt.check_operator_errors()


@pytest.mark.parametrize("rows", [1, 6, 33, 200])
@pytest.mark.parametrize("out", list(DTYPES))
def test_quantized_rows_as_input(tt, rows, out):
    g = torch.Generator().manual_seed(rows)
    spins = (torch.randint(0, 2, (rows, 777), generator=g) * 2 - 1).to(torch.int8)
    w = torch.randint(-128, 128, (90, 777), generator=g).to(torch.int8)
    sw = torch.rand(90, generator=g) + 0.5
    y = tt.int8_product(tt.QuantizedRows(spins.cuda()), tt.QuantizedRows(w.cuda(), sw.cuda()), out_dtype=DTYPES[out])
    check_product(y, spins.numpy().astype(np.int64), np.ones(rows, np.float32), w.numpy().astype(np.int64), sw.numpy(),
                  None, DTYPES[out])


@pytest.mark.parametrize("rows", [2, 40])
def test_strides_of_rows_and_output(tt, rows):
    K, N = 333, 95
    w = rand((N, K), torch.float32, 1)
    r = tt.quantize_rows(w.cuda())
    wq, sw = plain_quantize(w)
    big = rand((2 * rows, K + 9), torch.bfloat16, 2)
    x = big[::2, 3 : 3 + K]
    out = torch.full((rows, N + 13), 7.0, device="cuda")
    y = tt.int8_product(big.cuda()[::2, 3 : 3 + K], r, out=out[:, 5 : 5 + N])
    check_product(y, *plain_quantize(x), wq, sw, None, torch.float32)
    assert (out[:, :5] == 7).all() and (out[:, 5 + N :] == 7).all()  # beside the written columns: as they were
    xt = rand((K, rows), torch.float16, 3)  # columns in memory order
    check_product(tt.int8_product(xt.cuda().t(), r), *plain_quantize(xt.t()), wq, sw, None, torch.float16)
    x3 = rand((rows, 3, K), torch.float32, 4)
    y3 = tt.int8_product(x3.cuda(), r)
    assert y3.shape == (rows, 3, N)
    check_product(y3.reshape(-1, N), *plain_quantize(x3.reshape(-1, K)), wq, sw, None, torch.float32)


@pytest.mark.parametrize("rows", [1, 8, 9])
def test_largest_sums_are_exact(tt, rows):
    cols = 131071
    w = torch.full((3, cols), -128, dtype=torch.int8)
    x = torch.full((rows, cols), -128, dtype=torch.int8)
    w[1] = 127
    w[2, ::2] = 127
    y = tt.int8_product(tt.QuantizedRows(x.cuda()), tt.QuantizedRows(w.cuda(), torch.ones(3, device="cuda")))
    exact = x[:1].double() @ w.double().t()
    assert torch.equal(y.cpu(), exact.float().expand(rows, 3))


@pytest.mark.parametrize("rows", [3, 50])
def test_empty_rows_and_units(tt, rows):
    r = tt.quantize_rows(rand((4, 64), torch.float32, 1).cuda())
    assert tt.int8_product(torch.empty((0, 64), device="cuda"), r).shape == (0, 4)
    none = tt.QuantizedRows(torch.empty((0, 64), dtype=torch.int8, device="cuda"), torch.empty(0, device="cuda"))
    assert tt.int8_product(torch.ones((rows, 64), device="cuda"), none).shape == (rows, 0)
    assert tt.quantize_rows(torch.empty((0, 5), device="cuda")).shape == (0, 5)


@pytest.mark.parametrize("rows", [1, 70])
def test_captured_products_on_two_streams_and_graphs(tt, rows):
    K, N = 512, 200
    w = rand((N, K), torch.float32, 1)
    r = tt.quantize_rows(w.cuda())
    wq, sw = plain_quantize(w)
    xs = [rand((rows, K), torch.bfloat16, 10 + i) for i in range(2)]
    held = [x.cuda() for x in xs]
    tt.int8_product(held[0], r)
    graphs, outs = [], []
    for x in held:
        g = torch.cuda.CUDAGraph()
        with nat.capturing(g):
            outs.append(tt.int8_product(x, r))
        graphs.append(g)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in graphs]
    for _ in range(20):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    for x, y in zip(xs, outs):
        check_product(y, *plain_quantize(x), wq, sw, None, torch.bfloat16)


def test_refusals(tt):
    r = tt.quantize_rows(torch.ones((4, 64), device="cuda"))
    ok = torch.ones((2, 64), device="cuda")
    for args, kw, exc in [
        ((ok, torch.ones((4, 64))), {}, TypeError),
        ((ok.double(), r), {}, ValueError),
        ((ok.cpu(), r), {}, ValueError),
        ((ok[:, :63], r), {}, ValueError),
        ((ok, r), {"bias": torch.ones(5, device="cuda")}, ValueError),
        ((ok, r), {"bias": torch.ones(4, device="cuda", dtype=torch.float16)}, ValueError),
        ((ok, r), {"out_dtype": torch.int32}, ValueError),
        ((ok, r), {"out": torch.empty((3, 4), device="cuda")}, ValueError),
        ((ok, r), {"out": torch.empty((4, 2), device="cuda").t()}, ValueError),
        ((ok, r), {"out": torch.empty((1, 4), device="cuda").expand(2, 4)}, ValueError),
        ((ok[:, :4].contiguous(), tt.quantize_rows(torch.ones((4, 4), device="cuda"))), {"out": "x"}, ValueError),
        ((ok, tt.QuantizedRows(r.values)), {}, ValueError),
        ((ok.clone().requires_grad_(True), r), {}, RuntimeError),
    ]:
        if kw.get("out") is not None and isinstance(kw["out"], str):
            kw = {"out": args[0]}  # in place: read and written at the same time
        with pytest.raises(exc):
            tt.int8_product(*args, **kw)
    with torch.no_grad():
        tt.int8_product(ok.clone().requires_grad_(True), r)
    for bad in (torch.ones((2, 3)), torch.ones(3, device="cuda"), torch.ones((2, 3), device="cuda").double(),
                torch.ones((2, 0), device="cuda"), torch.ones((1, 131072), device="cuda")):
        with pytest.raises(ValueError):
            tt.quantize_rows(bad)
    for values, scale in ((torch.ones((2, 3), device="cuda"), None),
                          (torch.ones((2, 3), dtype=torch.int8, device="cuda"), torch.ones(3, device="cuda")),
                          (torch.ones((2, 3), dtype=torch.int8, device="cuda"), torch.ones(2))):
        with pytest.raises(ValueError):
            tt.QuantizedRows(values, scale)
