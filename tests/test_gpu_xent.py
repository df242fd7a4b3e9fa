"""Softmax cross entropy on the GPU against the formulas in 64 bits, with the errors of each step counted."""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


@pytest.fixture(scope="module")
def tt():
    import tt_thrml_b200

    return tt_thrml_b200


def batch(rows, k, v, dtype, seed, bias=True, ignored=0.1, scale=1.5):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape):
        return torch.randn(shape, generator=g, device="cuda")

    x, w = normal(rows, k).to(dtype), (normal(v, k) * (scale / math.sqrt(k))).to(dtype)
    y = torch.randint(0, v, (rows,), generator=g, device="cuda")
    if ignored:
        y = torch.where(torch.rand(rows, generator=g, device="cuda") < ignored, -100, y)
    return x, w, y, normal(v) * 0.5 if bias else None


def expected(x, w, y, bias, weight, ignore=-100):
    """Losses, gradients of sum weight * loss, and what each may be off by.

    Steps of float32 (u = 2^-24): a logit is a sum of ceil(K / 16) + 15 partial sums of exact products, each dropping at
    most 2 u of the sum of their magnitudes, and the bias (u).  A normaliser in the log2 domain: three roundings of its size,
    an exponential (2^-22 relative, 4 u more for its argument's rounding per unit of the argument), sums of V terms pairwise
    over at most V / 256 + 64 additions.  g is rounded to 16 bits; dx and dw are sums as the logits are and rounded once."""
    u = 2.0**-24
    K, V, T = x.shape[1], w.shape[0], x.shape[0]
    xd, wd = x.double(), w.double()
    l = xd @ wd.t()
    mag = xd.abs() @ wd.abs().t()
    if bias is not None:
        l = l + bias.double()
        mag = mag + torch.where(torch.isfinite(bias), bias.abs(), 0.0).double()
    dl = (math.ceil(K / 16) + 16) * 2 * u * mag
    z = torch.logsumexp(l, 1)
    possible = torch.isfinite(z)
    zs = torch.where(possible, z, 0.0)
    counts = (y != ignore) & possible
    at = torch.where(y == ignore, 0, y)
    off = dl.amax(1)
    spread = 1.0 + zs.abs() + torch.where(torch.isfinite(l), l, 0.0).abs().amax(1)
    dz = off + (V / 256 + 64 + 16) * u + 12 * u * spread
    ly = l.gather(1, at[:, None])[:, 0]
    loss = torch.where(y == ignore, 0.0, torch.where(possible, z - ly, math.inf))
    dloss = torch.where(y == ignore, 0.0, dz + off + 2 * u * spread)
    p = torch.where(possible[:, None], torch.exp(l - zs[:, None]), 0.0)
    r = torch.where(counts, weight.double(), 0.0)[:, None]
    hit = torch.zeros_like(p).scatter_(1, at[:, None], 1.0)
    g = r * (p - hit)
    half = torch.finfo(x.dtype).eps / 2
    dg0 = r.abs() * (p * (dl + (dz + 12 * u * spread)[:, None]) + 4 * u * (p + hit))  # before its rounding
    # float16 holds g as 2^14 g / (the largest weight): its smallest step is 2^-24 of that
    tiny = 2.0**-25 * 2.0**-14 * float(r.abs().max()) if x.dtype == torch.float16 else 0.0
    few = x.shape[0] <= 128  # g in two pieces: the rounding of the second one, 16 bits further down
    dg = dg0 + (half * half if few else half) * g.abs() + torch.where(r != 0, tiny, 0.0)

    def product(a, da, b, n):
        exact = a @ b
        err = da @ b.abs() + (math.ceil(n / 16) + 40) * 2 * u * ((a.abs() + da) @ b.abs())
        step = float(torch.finfo(x.dtype).smallest_normal) * torch.finfo(x.dtype).eps
        return exact, err + half * (exact.abs() + err) + step

    dx = product(g, dg, wd, V)
    dw = product(g.t(), dg.t(), xd, T)
    db = g.sum(0), dg0.sum(0) + (T + 8) * u * (g.abs() + dg0).sum(0)
    return (loss, dloss), dx, dw, db


def close(name, got, want):
    exact, tol = want
    got = got.double()
    inf = torch.isinf(exact)
    assert torch.equal(got[inf], exact[inf]), name
    bad = ~((got - exact).abs() <= tol) & ~inf
    assert not bad.any(), (name, int(bad.sum()), float(((got - exact).abs() - tol)[bad].max()), float(exact[~inf].abs().max()))


def check(tt, x, w, y, bias, reduction, ignore=-100, rows_grad=None):
    leaves = [t.clone().requires_grad_(True) for t in (x, w)]
    b = None if bias is None else bias.clone().requires_grad_(True)
    loss = tt.softmax_cross_entropy(*leaves, y, bias=b, reduction=reduction, ignore_index=ignore)
    n = max(1, int((y != ignore).sum()))
    if reduction == "none":
        weight = torch.linspace(-1, 2, x.shape[0], device="cuda") if rows_grad is None else rows_grad
    else:
        weight = torch.full((x.shape[0],), 1.0 / n if reduction == "mean" else 1.0, device="cuda")
    want, dx, dw, db = expected(x, w, y, bias, weight, ignore)
    loss.backward(weight if reduction == "none" else None)
    if reduction == "none":
        close("loss", loss, want)
    else:
        factor = 1.0 / n if reduction == "mean" else 1.0
        total = want[0].sum() * factor
        close("loss", loss, (total, want[1].sum() * factor + 2.0**-22 * total.abs()))
    close("dx", leaves[0].grad, dx)
    close("dw", leaves[1].grad, dw)
    if bias is not None:
        close("db", b.grad, db)
    tt.check_operator_errors()


SIZES = [(1, 8, 2), (1, 1, 1), (3, 5, 7), (1, 512, 1000), (31, 64, 33), (33, 72, 257), (128, 129, 255), (129, 200, 640),
         (257, 65, 1031), (300, 1001, 5003), (700, 96, 70), (1500, 24, 3)]


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("rows,k,v", SIZES)
def test_losses_and_gradients(tt, rows, k, v, dtype):
    x, w, y, bias = batch(rows, k, v, DTYPES[dtype], rows + k + v)
    check(tt, x, w, y, bias, "mean")


@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("with_bias", [False, True])
def test_reductions(tt, reduction, dtype, with_bias):
    x, w, y, bias = batch(200, 136, 777, DTYPES[dtype], 5, bias=with_bias)
    check(tt, x, w, y, bias, reduction)


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("rows,k,v", [(16500, 40, 8700), (9000, 257, 16001)])
def test_categories_in_several_pieces(tt, rows, k, v, dtype):
    """More than 256 MiB of differences: the gradients of x are sums over pieces of the categories."""
    x, w, y, bias = batch(rows, k, v, DTYPES[dtype], 3)
    check(tt, x, w, y, bias, "mean")


@pytest.mark.parametrize("rows,k,v", [(4000, 2048, 6000), (2500, 1000, 9000)])
def test_many_tiles(tt, rows, k, v):
    x, w, y, bias = batch(rows, k, v, torch.bfloat16, 4, bias=k == 1000)
    check(tt, x, w, y, bias, "mean")
