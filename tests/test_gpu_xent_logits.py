"""Rows that are predicted well: their differences are what is left of probabilities near 1, so the logits of the backward pass
have to be those that the normalisers were made of, whichever gradients are asked for."""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
U = 2.0**-24


@pytest.fixture(scope="module")
def tt():
    import tt_thrml_b200

    return tt_thrml_b200


def confident(rows, k, v, dtype, seed):
    """Rows whose target's logit is 10.5 to 20.5 (losses of about v e^-logit) and whose other logits are small: x has the signs
    of its target's weights, so that every product of the target's logit is positive."""
    g = torch.Generator(device="cuda").manual_seed(seed)

    def magnitudes(*shape):
        return 0.5 + 0.5 * torch.rand(shape, generator=g, device="cuda")

    w = torch.where(torch.rand(v, k, generator=g, device="cuda") < 0.5, -1.0, 1.0) * magnitudes(v, k) / 8
    y = torch.randint(0, v, (rows,), generator=g, device="cuda")
    x = torch.sign(w[y]) * magnitudes(rows, k)
    logit = torch.linspace(10.5, 20.5, rows, device="cuda") if rows > 1 else torch.full((1,), 15.0, device="cuda")
    x = x * (logit / (x * w[y]).sum(1))[:, None]
    return x.to(dtype), w.to(dtype), y, torch.randn(v, generator=g, device="cuda") * 0.1


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("with_bias", [False, True], ids=["no bias", "bias kept"])
@pytest.mark.parametrize("rows,k,v", [(40, 2048, 512), (300, 4096, 500), (300, 16384, 512), (100, 16384, 60), (700, 8192, 33)])
def test_gradients_of_confident_rows(tt, rows, k, v, with_bias, dtype):
    """Bounds, with u = 2^-24.  A logit is summed in pieces of at most 512 columns: 32 additions of 16 products and 15 inside an
    addition, each dropping at most 2 u of the piece's magnitudes; the pieces, of at least 128 columns, are added in float32: k / 128
    additions; the bias u.  These errors E are the same in both passes: they change a difference p - 1 and a loss by at most
    2 E (1 - p), another probability by 2 E p.  Beside that probabilities and sums of exponentials are off by 2^-22 each,
    (v / 256 + 64) additions and 40 u for arguments of up to 30 in the log2 domain."""
    x, w, y, bias = confident(rows, k, v, DTYPES[dtype], rows + k)
    b = bias if with_bias else None  # a bias, but not its gradient
    leaves = [t.clone().requires_grad_(True) for t in (x, w)]
    loss = tt.softmax_cross_entropy(*leaves, y, bias=b, reduction="none")
    dx, dw = torch.autograd.grad(loss.sum(), leaves)

    xd, wd = x.double(), w.double()
    logits = xd @ wd.t() + (0.0 if b is None else b.double())
    mag = xd.abs() @ wd.abs().t()
    E = ((2 * 47 + k / 128) * U * mag + U * logits.abs()).amax(1)
    relative = 2 * 2.0**-22 + (v / 256 + 64 + 40) * U
    z = torch.logsumexp(logits, 1)
    at = torch.arange(rows, device="cuda")
    exact = z - logits[at, y]
    assert float(exact.min()) < 1e-5 and float(exact.max()) > 5e-4
    assert ((loss.double() - exact).abs() <= 2 * E * exact + relative + U * exact).all()
    p = torch.exp(logits - z[:, None])
    g = p.clone()
    g[at, y] = torch.expm1(-exact)
    off = (2 * E[:, None] + relative + 2 * U) * p
    off[at, y] = 2 * E * -g[at, y] + relative + 2 * U
    half = torch.finfo(x.dtype).eps / 2
    few = rows <= 128 or v <= 64  # held in two pieces
    # float16 holds 2^14 g in steps of at least 2^-24
    dg = off + (half * half if few else half) * (g.abs() + off) + (2.0**-39 if x.dtype == torch.float16 else 0.0)

    def close(name, got, a, da, c, n):
        want = a @ c
        tol = da @ c.abs() + (math.ceil(n / 16) + 40) * 2 * U * ((a.abs() + da) @ c.abs())
        tol = tol + half * (want.abs() + tol) + float(torch.finfo(x.dtype).smallest_normal) * torch.finfo(x.dtype).eps
        bad = (got.double() - want).abs() > tol
        assert not bad.any(), (name, int(bad.sum()), float(((got.double() - want).abs() / tol).max()))

    close("dx", dx, g, dg, wd, v)
    close("dw", dw, g.t(), dg.t(), xd, rows)
    tt.check_operator_errors()


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("rows,k,v", [(1, 512, 1000), (40, 2048, 512), (90, 40, 200), (129, 200, 640), (300, 4096, 5003), (700, 8192, 33),
                                      (100, 16384, 60), (3000, 1024, 9000), (16500, 600, 8700)])
def test_gradients_do_not_depend_on_which_are_asked_for(tt, rows, k, v, dtype):
    """The gradients of x and w are the same bits with and without that of the bias, and without a bias those of zeros."""
    x, w, y, bias = confident(rows, k, v, DTYPES[dtype], 1)

    def grads(b, *names):
        t = {n: s.clone().requires_grad_(n in names) for n, s in (("x", x), ("w", w))}
        if b is not None:
            t["b"] = b.clone().requires_grad_("b" in names)
        loss = tt.softmax_cross_entropy(t["x"], t["w"], y, bias=t.get("b"))
        return dict(zip(names, torch.autograd.grad(loss, [t[n] for n in names])))

    every = grads(bias, "x", "w", "b")
    for names in (("x", "w"), ("x",), ("w",), ("x", "b"), ("w", "b")):
        for n, g in grads(bias, *names).items():
            assert torch.equal(g, every[n]), (names, n)
    zeros, none = grads(torch.zeros_like(bias), "x", "w"), grads(None, "x", "w")
    assert torch.equal(zeros["x"], none["x"]) and torch.equal(zeros["w"], none["w"])
    tt.check_operator_errors()
