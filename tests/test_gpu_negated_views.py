"""Operators on negated views (the imaginary part of a conjugate is one): the values are those that the view shows."""

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def tt():
    import tt_thrml_b200

    return tt_thrml_b200


def negated(t):
    """A view of memory that holds -t."""
    view = torch._neg_view(-t)
    assert view.is_neg() and torch.equal(view, t)
    return view


@pytest.mark.parametrize("cols", [1, 40, 41])
def test_cross_entropy(tt, cols):
    g = torch.Generator(device="cuda").manual_seed(1)
    x, w = (torch.randn(n, cols, generator=g, device="cuda").bfloat16() for n in (50, 70))
    bias, grad = torch.randn(70, generator=g, device="cuda"), torch.randn(50, generator=g, device="cuda")
    y = torch.randint(0, 70, (50,), generator=g, device="cuda")

    def run(of):
        leaves = [of(t).requires_grad_(True) for t in (x.clone(), w.clone(), bias.clone())]
        loss = tt.softmax_cross_entropy(leaves[0], leaves[1], of(y), bias=leaves[2], reduction="none")
        return loss, *torch.autograd.grad(loss, leaves, of(grad))

    for a, b in zip(run(negated), run(lambda t: t)):
        assert torch.equal(a, b)
    a, b = (tt.CategoricalReadout(cols, 70, seed=1) for _ in range(2))
    assert torch.equal(a.step(negated(x), y), b.step(x, y)) and torch.equal(a.weights, b.weights)


@pytest.mark.parametrize("shape", [(7,), (33, 41)])
def test_dropout(tt, shape):
    x, grad = torch.randn(shape, device="cuda"), torch.randn(shape, device="cuda")

    def run(of):
        leaf = of(x.clone()).requires_grad_(True)
        y = tt.dropout(leaf, 0.3, seed=5)
        return y, *torch.autograd.grad(y, leaf, of(grad))

    for a, b in zip(run(negated), run(lambda t: t)):
        assert torch.equal(a, b)


@pytest.mark.parametrize("rows", [1, 3, 50])
@pytest.mark.parametrize("cols", [1, 40, 41])
def test_4_bit_rows(tt, rows, cols):
    g = torch.Generator(device="cuda").manual_seed(2)
    x, w, bias = (torch.randn(*s, generator=g, device="cuda") for s in ((rows, cols), (60, cols), (60,)))
    q = tt.quantize_fp4(w)
    assert torch.equal(tt.quantize_fp4(negated(x)).dequantize(), tt.quantize_fp4(x).dequantize())
    assert torch.equal(tt.fp4_product(negated(x), q, bias=negated(bias)), tt.fp4_product(x, q, bias=bias))
    given = tt.Fp4Rows(q.codes, q.block_scale, negated(q.scale), cols=cols)
    assert torch.equal(given.dequantize(), q.dequantize())
    with pytest.raises(ValueError, match="negated"):
        tt.fp4_product(x, q, out=negated(torch.zeros(rows, 60, device="cuda")))
