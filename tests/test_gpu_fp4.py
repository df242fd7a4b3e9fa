"""4-bit floating point rows and products on the GPU against a plain implementation in 64 bits."""

import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
U = 2.0**-24  # half a step of float32, relative
GRID = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])


@pytest.fixture(scope="module")
def tt():
    import tt_thrml_b200

    return tt_thrml_b200


def nearest_e2m1(y):
    """Index of the nearest code's magnitude, ties to the even index, from float32 values."""
    a = np.abs(y).astype(np.float64)
    mids = (GRID[1:] + GRID[:-1]) / 2
    down = np.searchsorted(mids, a, side="left")  # a tie stays below
    up = np.searchsorted(mids, a, side="right")
    return np.where(down % 2 == 0, down, up)


def plain_quantize(x):
    """(signed code values, block scales, row scales) of the rows of a CPU tensor, decided in float32."""
    f = x.float().numpy()
    rows, cols = f.shape
    with np.errstate(all="ignore"):
        top = np.abs(f).max(1)
        finite = np.isfinite(top)
        live = finite & (top >= np.float32(2.0**-100))
        inv = np.zeros_like(top)
        inv[live] = np.float32(2688.0) / top[live]
        scale = np.where(live, top * np.float32(1.0 / 2688.0), np.where(finite, np.float32(0.0), np.float32(np.nan)))
        blocks = -(-cols // 16)
        pad = np.zeros((rows, blocks * 16), np.float32)
        pad[:, :cols] = f
        b = pad.reshape(rows, blocks, 16)
        t = (np.abs(b).max(2) * inv[:, None]) * np.float32(1.0 / 6.0)
        e = torch.from_numpy(np.minimum(t, np.float32(448.0))).to(torch.float8_e4m3fn).float().numpy()
        factor = np.where(e > 0, inv[:, None] / np.where(e > 0, e, np.float32(1.0)), np.float32(0.0)).astype(np.float32)
        y = b * factor[:, :, None]
        codes = np.copysign(GRID[nearest_e2m1(y)], y).reshape(rows, -1)[:, :cols]
    return codes, e, scale


def rand(shape, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(shape, generator=g).to(dtype)


def unpacked(q):
    """Code values of Fp4Rows as float64 [rows, cols]."""
    c = q.codes.cpu().numpy()
    both = np.stack([c & 15, c >> 4], 2).reshape(c.shape[0], -1)[:, : q.cols]
    return np.where(both >= 8, -GRID[both & 7], GRID[both & 7])


SHAPES = [(1, 1), (3, 15), (8, 16), (5, 17), (33, 1000), (7, 1024), (9, 1025), (2, 4103), (4, 8192), (130, 300), (1, 40000)]


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("rows,cols", SHAPES)
def test_quantize_matches_the_formula(tt, rows, cols, dtype):
    x = rand((rows, cols), DTYPES[dtype], rows * 7 + cols)
    q = tt.quantize_fp4(x.cuda())
    codes, blocks, scale = plain_quantize(x)
    assert np.array_equal(q.scale.cpu().numpy(), scale)
    assert np.array_equal(q.block_scale.float().cpu().numpy(), blocks)
    assert np.array_equal(unpacked(q), codes)
    values = (codes * np.repeat(blocks, 16, 1)[:, :cols]).astype(np.float32) * scale[:, None]
    assert np.array_equal(q.dequantize().cpu().numpy(), values)
    again = tt.Fp4Rows(q.codes.clone(), q.block_scale, q.scale, cols=cols)
    assert torch.equal(again.blocks, q.blocks) and torch.equal(again.dequantize(), q.dequantize())


def check_product(y, a, sa, b, sb, bias, dtype):
    """|y - exact| within: partial sums of at most 16 exact products, each addition dropping at most 2 U of the sum of the
    magnitudes; the product of the scales, the scaling and the bias addition (U each); the rounding to the output type."""
    k = a.shape[1]
    s = np.outer(sa.astype(np.float64), sb.astype(np.float64))
    prod = (a @ b.T) * s
    mag = (np.abs(a) @ np.abs(b).T) * s
    exact = prod if bias is None else prod + bias.astype(np.float64)
    tol = (math.ceil(k / 16) + 16) * 2 * U * mag + 3 * U * np.abs(prod) + U * np.abs(exact)
    if dtype != torch.float32:
        tol = tol + torch.finfo(dtype).eps / 2 * (np.abs(exact) + tol)
    tol = tol + float(torch.finfo(dtype).smallest_normal) * torch.finfo(dtype).eps
    got = y.double().cpu().numpy()
    assert got.shape == exact.shape
    bad = ~(np.abs(got - exact) <= tol)
    assert not bad.any(), (int(bad.sum()), float(np.abs(got - exact).max()), float(tol.max()))


def with_blocks(codes, blocks):
    return codes * np.repeat(blocks, 16, 1)[:, : codes.shape[1]].astype(np.float64)


def run_product(tt, m, n, k, dtype, bias, seed):
    x, w = rand((m, k), DTYPES[dtype], seed), rand((n, k), torch.float32, seed + 1)
    # blocks of very different sizes, so that a scale in the wrong place shows
    w = w * torch.exp2(torch.randint(-6, 1, (n, -(-k // 16)), generator=torch.Generator().manual_seed(seed + 2)).float()
                       ).repeat_interleave(16, 1)[:, :k]
    x = (x.float() * torch.exp2(torch.randint(-6, 1, (m, -(-k // 16)), generator=torch.Generator().manual_seed(seed + 3)).float()
                                ).repeat_interleave(16, 1)[:, :k]).to(DTYPES[dtype])
    b = rand((n,), torch.float32, seed + 4) if bias else None
    y = tt.fp4_product(x.cuda(), tt.quantize_fp4(w.cuda()), bias=None if b is None else b.cuda())
    (ca, ba, sa), (cb, bb, sb) = plain_quantize(x), plain_quantize(w)
    check_product(y, with_blocks(ca, ba), sa, with_blocks(cb, bb), sb, None if b is None else b.numpy(), DTYPES[dtype])
    tt.check_operator_errors()


@pytest.mark.parametrize("m,n,k", [(16, 64, 64), (128, 64, 256), (128, 128, 256), (128, 192, 512), (20, 300, 40), (37, 2047, 501),
                                   (130, 33, 1000), (200, 700, 4100), (129, 257, 8192), (1, 1, 1), (1, 500, 1000), (2, 64, 33),
                                   (300, 1000, 300), (5, 5000, 2048)])
@pytest.mark.parametrize("dtype", list(DTYPES))
def test_products(tt, m, n, k, dtype):
    run_product(tt, m, n, k, dtype, (m + n) % 2 == 0, m + n + k)


@pytest.mark.parametrize("m,n,k", [(4100, 4203, 600), (2560, 5120, 1280), (8192, 300, 257)])
def test_products_of_many_tiles(tt, m, n, k):
    run_product(tt, m, n, k, "bf16", True, 3)


@pytest.mark.parametrize("m", [1, 2, 3, 4])
@pytest.mark.parametrize("n,k", [(1, 1), (130, 16), (257, 1000), (1000, 1024), (2048, 4096), (300, 4097), (129, 9001), (19000, 500)])
def test_products_of_few_rows(tt, m, n, k):
    for dtype in DTYPES:
        run_product(tt, m, n, k, dtype, n % 2 == 0, m + n + k)


def test_special_rows(tt):
    """Zeros, tiny and huge magnitudes, infinities and NaN; a row that is not finite is NaN in its own products alone."""
    x = rand((9, 200), torch.float32, 5)
    x[1] = 0
    x[2] *= 2.0**-104  # below 2^-100: zeros
    x[3] *= 2.0**-90
    x[4] *= 2.0**120
    x[5, 7] = math.inf
    x[6, 199] = math.nan
    x[7] = 0
    x[7, 31] = -3.0
    q = tt.quantize_fp4(x.cuda())
    codes, blocks, scale = plain_quantize(x)
    assert np.array_equal(q.scale.cpu().numpy(), scale, equal_nan=True) and scale[1] == scale[2] == 0
    fine = [0, 1, 2, 3, 4, 7, 8]
    assert np.array_equal(unpacked(q)[fine], codes[fine])
    assert np.array_equal(q.block_scale.float().cpu().numpy()[fine], blocks[fine])
    values = q.dequantize().cpu()
    # code and block are the largest, 6 * 448; three roundings: of 1 / 2688, of the row's scale, of the value
    assert abs(values[7, 31] + 3.0) <= 3 * 3.0 * U and torch.count_nonzero(values[7]) == 1
    assert torch.isnan(values[5]).all() and torch.isnan(values[6]).all() and torch.isfinite(values[fine]).all()
    w = tt.quantize_fp4(rand((300, 200), torch.float32, 6).cuda())
    for rows in (slice(0, 9), slice(4, 8)):  # through the tiles, and as few rows
        y = tt.fp4_product(x[rows].cuda(), w)
        bad = torch.isnan(y).all(1).cpu()
        assert bad.tolist() == [i in (5, 6) for i in range(9)][rows] and torch.isfinite(y[~bad.cuda()]).all()
    y = tt.fp4_product(rand((150, 200), torch.float32, 7).cuda(), q)  # weights that are not finite: their units alone
    assert torch.isnan(y[:, [5, 6]]).all() and torch.isfinite(y[:, fine]).all()
    tt.check_operator_errors()


def test_spins_are_their_own_codes(tt):
    """Rows of +-1 are exact in 4 bits, so fields of spins are exact products with the weights' values."""
    s = torch.where(rand((70, 96), torch.float32, 8) > 0, 1.0, -1.0).bfloat16().cuda()
    q = tt.quantize_fp4(s)
    exact = q.dequantize()
    assert ((exact - s.float()).abs() <= 3 * U).all()  # 2688 fl(fl(1 / 2688) 1): of 1 / 2688, the row's scale and the value


@pytest.mark.parametrize("m", [1, 4, 6, 150])
@pytest.mark.parametrize("layout", ["sliced", "shifted", "odd pitch", "transposed", "expanded", "three dimensions"])
def test_strides_and_shapes(tt, m, layout):
    x = rand((m, 136), torch.bfloat16, 9).cuda()
    w = tt.quantize_fp4(rand((200, 136), torch.float32, 10).cuda())
    want = tt.fp4_product(x, w)
    if layout == "sliced":
        y = torch.empty(m, 300, dtype=x.dtype, device="cuda")[:, 8:144].copy_(x)
    elif layout == "shifted":
        y = torch.empty(m * 136 + 1, dtype=x.dtype, device="cuda")[1:].view(m, 136).copy_(x)
    elif layout == "odd pitch":
        y = torch.empty(m, 139, dtype=x.dtype, device="cuda")[:, :136].copy_(x)
    elif layout == "transposed":
        y = x.t().contiguous().t()
    elif layout == "expanded":
        y = x[:1].expand(m, 136)
        want = want[:1].expand(m, 200)
    else:
        y, want = x.view(m, 1, 136), want.view(m, 1, 200)
    assert torch.equal(tt.fp4_product(y, w), want)
    if y.dim() == 2:
        assert torch.equal(tt.quantize_fp4(y).dequantize(), tt.quantize_fp4(y.contiguous()).dequantize())
    out = torch.full((m, 264), 7.0, dtype=torch.float32, device="cuda")
    got = tt.fp4_product(y, w, out=out[:, 3:203].view(*y.shape[:-1], 200) if y.dim() == 2 else out[:, 3:203].unsqueeze(1))
    assert torch.equal(got.to(x.dtype), want)
    assert (out[:, :3] == 7).all() and (out[:, 203:] == 7).all()  # what lies beside is left alone


def test_quantized_rows_multiply_as_floats_do(tt):
    for m in (5, 140, 1000):
        x, w = rand((m, 700), torch.bfloat16, m).cuda(), tt.quantize_fp4(rand((260, 700), torch.float32, 3).cuda())
        bias = rand((260,), torch.float32, 4).cuda()
        a = tt.fp4_product(tt.quantize_fp4(x), w, bias=bias)
        assert a.dtype == torch.float32 and torch.equal(a, tt.fp4_product(x, w, bias=bias, out_dtype=torch.float32))
    few = tt.fp4_product(tt.quantize_fp4(x[:2]), w, bias=bias)  # two rows: another kernel, other sums
    torch.testing.assert_close(few, tt.fp4_product(x[:2], w, bias=bias, out_dtype=torch.float32), rtol=1e-5, atol=1e-4)


def test_given_codes_with_odd_rows(tt):
    """Rows of codes as a checkpoint holds them: odd columns, unaligned pitch, a stray code behind the last column."""
    codes = torch.randint(0, 256, (130, 21), generator=torch.Generator().manual_seed(1), dtype=torch.uint8)
    blocks = (torch.rand(130, 3, generator=torch.Generator().manual_seed(2)) * 400).to(torch.float8_e4m3fn)
    scale = torch.rand(130, generator=torch.Generator().manual_seed(3)) + 0.1
    q = tt.Fp4Rows(codes.cuda(), blocks.cuda(), scale.cuda(), cols=41)
    both = np.stack([codes.numpy() & 15, codes.numpy() >> 4], 2).reshape(130, -1)[:, :41]
    c = np.where(both >= 8, -GRID[both & 7], GRID[both & 7]) * np.repeat(blocks.float().numpy(), 16, 1)[:, :41]
    assert np.array_equal(q.dequantize().cpu().numpy(), c.astype(np.float32) * scale.numpy()[:, None])
    for m in (3, 200):
        x = rand((m, 41), torch.float32, m)
        ca, ba, sa = plain_quantize(x)
        check_product(tt.fp4_product(x.cuda(), q), with_blocks(ca, ba), sa, c, scale.numpy(), None, torch.float32)


@pytest.mark.parametrize("m", [1, 3, 70, 300])
@pytest.mark.parametrize("cols", [1, 33, 255])
def test_the_half_byte_behind_odd_columns_does_not_count(tt, m, cols):
    """Codes whose last half byte holds anything, on both sides of a product: the sums are those of the columns."""
    g = torch.Generator().manual_seed(cols + m)
    bytes_, blocks = (cols + 1) // 2, (cols + 15) // 16

    def rows(n):
        codes = torch.randint(0, 256, (n, (bytes_ + 15) // 16 * 16), generator=g, dtype=torch.uint8).cuda()[:, :bytes_]
        codes[:, -1] |= 0x70
        return tt.Fp4Rows(codes, torch.full((n, blocks), 2.0).to(torch.float8_e4m3fn).cuda(), torch.ones(n).cuda(), cols=cols)

    x, w = rows(m), rows(90)
    exact = x.dequantize().double() @ w.dequantize().double().t()
    assert torch.equal(tt.fp4_product(x, w).double(), exact)  # sums of multiples of 1 below 255 * 144: exact in float32
    assert x.codes.shape == (m, bytes_) and int((x.codes[:, -1] >> 4).max()) == 0


def test_nothing_to_do(tt):
    w = tt.quantize_fp4(torch.ones(4, 32, device="cuda"))
    assert tt.fp4_product(torch.ones(0, 32, device="cuda"), w).shape == (0, 4)
    e = tt.quantize_fp4(torch.ones(0, 32, device="cuda"))
    assert e.shape == (0, 32) and e.dequantize().shape == (0, 32)
    assert tt.fp4_product(torch.ones(3, 32, device="cuda"), e).shape == (3, 0)


def test_captured_products_replay(tt):
    w = tt.quantize_fp4(rand((300, 256), torch.float32, 1).cuda())
    for m in (2, 64, 400):
        x = rand((m, 256), torch.bfloat16, m).cuda()
        tt.fp4_product(x, w)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.stream(side), torch.cuda.graph(graph, stream=side):
            y = tt.fp4_product(x, w)
            q = tt.quantize_fp4(x).dequantize()
        for seed in range(2):
            x.copy_(rand((m, 256), torch.bfloat16, 100 + seed))
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(y, tt.fp4_product(x, w)) and torch.equal(q, tt.quantize_fp4(x).dequantize())


def test_rows_of_more_than_2_to_the_32_elements(tt):
    rows, cols = 70_000, 65_536
    x = torch.empty(rows, cols, dtype=torch.bfloat16, device="cuda")
    g = torch.Generator(device="cuda").manual_seed(1)
    for at in range(0, rows, 10_000):
        x[at : at + 10_000] = torch.randn(10_000, cols, generator=g, device="cuda")
    q = tt.quantize_fp4(x)
    for at in (0, 32_768, rows - 130):
        part = tt.quantize_fp4(x[at : at + 130].clone())
        assert torch.equal(part.codes, q.codes[at : at + 130]) and torch.equal(part.scale, q.scale[at : at + 130])
    y = x[5:15].clone()
    del x
    big = tt.fp4_product(y, q)
    assert torch.equal(big[:, -130:], tt.fp4_product(y, part))
    tt.check_operator_errors()


def test_refusals(tt):
    x = torch.ones(3, 32, device="cuda")
    w = tt.quantize_fp4(x)
    scale = torch.ones(3, device="cuda")
    blocks = w.block_scale
    for args, kw, match in [
        ((x, w.codes), {}, "must be Fp4Rows"), ((x[:, :30], w), {}, "columns"), ((x.double(), w), {}, "float32, bfloat16"),
        ((x, w), {"bias": torch.ones(4, device="cuda")}, "bias must be"), ((x, w), {"out_dtype": torch.int32}, "out_dtype"),
        ((x, w), {"out": torch.ones(3, 4, device="cuda")}, "out must be"), ((x, w), {"out": x[:, :3]}, "shares memory"),
        ((x, w), {"out": torch.ones(1, 3, device="cuda").expand(3, 3)}, "dense rows"), ((x.cpu(), w), {}, "CUDA device"),
        ((x.clone().requires_grad_(True), w), {}, "4-bit products have no backward"),
    ]:
        with pytest.raises((ValueError, TypeError, RuntimeError), match=match):
            tt.fp4_product(*args, **kw)
    with pytest.raises(RuntimeError, match="no backward"):
        tt.quantize_fp4(x.clone().requires_grad_(True))
    for bad, match in [(x.int(), "float32"), (x[0], "matrix"), (torch.ones(2, 0, device="cuda"), "columns"), (x.cpu(), "CUDA")]:
        with pytest.raises(ValueError, match=match):
            tt.quantize_fp4(bad)
    for args, kw, match in [
        ((w.codes.int(), blocks, scale), {}, "uint8"), ((w.codes, blocks[:, :1], scale), {}, "block_scale"),
        ((w.codes, blocks.float(), scale), {}, "float8_e4m3fn"), ((w.codes, blocks, scale[:2]), {}, "scale must be"),
        ((w.codes, blocks, scale), {"cols": 30}, "bytes of codes"), ((w.codes.cpu(), blocks, scale), {}, "CUDA"),
    ]:
        with pytest.raises(ValueError, match=match):
            tt.Fp4Rows(*args, **kw)
    w.scale.requires_grad_(True)
    with pytest.raises(RuntimeError, match="scale of weights"):
        tt.fp4_product(x, w)
