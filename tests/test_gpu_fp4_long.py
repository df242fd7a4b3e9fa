"""Products of 4-bit rows with long sums, against 64 bits."""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0**-24


@pytest.fixture(scope="module")
def tt():
    import tt_thrml_b200

    return tt_thrml_b200


@pytest.mark.parametrize("signs", ["both", "one"])
@pytest.mark.parametrize("m,n,k", [(1, 130, 32768), (4, 70, 32001), (3, 64, 32769), (130, 70, 65536), (300, 300, 1 << 20), (5, 64, (1 << 20) - 1),
                                   (1500, 2100, 40000)])
def test_long_sums(tt, m, n, k, signs):
    """Partial sums of at most 16 exact products, each addition dropping at most 2 u of the sum of the magnitudes; the rows'
    scales and their product (u each)."""
    g = torch.Generator(device="cuda").manual_seed(m + n)
    x, w = (torch.randn(r, k, generator=g, device="cuda") for r in (m, n))
    if signs == "one":
        x, w = x.abs(), w.abs()
    w4 = tt.quantize_fp4(w)
    y = tt.fp4_product(x, w4, out_dtype=torch.float32)
    rows = [0, m - 1, m // 2, m // 3]
    # codes times blocks are exact in float32; the rows' scales go on at the end, as in the kernel
    x4, w4r = tt.quantize_fp4(x[rows]), tt.quantize_fp4(w)
    one_x, one_w = (tt.Fp4Rows(q.codes, q.block_scale, torch.ones_like(q.scale), cols=k).dequantize().double() for q in (x4, w4r))
    scale = torch.outer(x4.scale.double(), w4.scale.double())
    exact, mag = (one_x @ one_w.t()) * scale, (one_x.abs() @ one_w.abs().t()) * scale
    tol = (math.ceil(k / 16) + 16) * 2 * U * mag + 3 * U * exact.abs()
    assert ((y[rows].double() - exact).abs() <= tol).all()
    if signs == "both":  # nothing adds up where the signs differ
        assert float((y[rows].double() - exact).norm()) <= 2.0**-21 * float(exact.norm())
    tt.check_operator_errors()
