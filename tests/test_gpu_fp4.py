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
