"""Calls of the categorical readout in orders that the documentation allows."""

import pytest
import torch

from test_gpu_readout import data

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def tt():
    import tt_thrml_b200

    return tt_thrml_b200


def test_a_refused_step_changes_nothing(tt):
    """Neither weights nor masks of the steps after it."""
    x, y = data(64, 48, 30, 1)
    a, b = (tt.CategoricalReadout(48, 30, dropout=0.5, seed=6, lr=1e-2) for _ in range(2))
    for step in range(3):
        with pytest.raises(ValueError, match="targets"):
            a.step(x, y[:-1])
        with pytest.raises(ValueError, match="columns"):
            a.step(x[:, :-1], y)
        assert torch.equal(a.step(x, y), b.step(x, y)), step
        assert torch.equal(a.weights, b.weights) and torch.equal(a.bias, b.bias)


def test_fields_are_those_of_the_last_quantize(tt):
    """Weights and bias of one time: steps after quantize() do not show before the next one."""
    x, y = data(64, 48, 30, 2)
    r = tt.CategoricalReadout(48, 30, seed=7, lr=1e-1)
    r.step(x, y)
    r.quantize()
    fields, bias = r.fields(x), r.bias.clone()
    r.step(x, y)
    assert not torch.equal(r.bias, bias)
    assert torch.equal(r.fields(x), fields)
    assert torch.equal(fields, tt.fp4_product(x, r.served, bias=bias))
    r.quantize()
    assert torch.equal(r.fields(x), tt.fp4_product(x, tt.quantize_fp4(r.weights), bias=r.bias))


@pytest.mark.parametrize("kind", [torch.bfloat16, torch.float16, torch.float64])
def test_another_default_dtype(tt, kind):
    """The masters are float32 and the same numbers, whatever type new tensors have by default."""
    x, y = data(64, 48, 30, 3)
    want = tt.CategoricalReadout(48, 30, dropout=0.2, seed=8)
    loss = want.step(x, y)
    was = torch.get_default_dtype()
    torch.set_default_dtype(kind)
    try:
        r = tt.CategoricalReadout(48, 30, dropout=0.2, seed=8)
        assert torch.equal(r.step(x, y), loss)
        r.quantize()
        fields = r.fields(x)
    finally:
        torch.set_default_dtype(was)
    assert r.weights.dtype == r.bias.dtype == r.gradient[0].dtype == torch.float32
    assert torch.equal(r.weights, want.weights)
    want.quantize()
    assert torch.equal(fields, want.fields(x))


def test_values_of_4_bit_rows_have_no_gradient(tt):
    """As products with such rows do, their values refuse a scale that requires one instead of dropping it."""
    q = tt.quantize_fp4(torch.ones(4, 32, device="cuda"))
    given = tt.Fp4Rows(q.codes, q.block_scale, q.scale.clone().requires_grad_(True), cols=32)
    with pytest.raises(RuntimeError, match="scale requires a gradient"):
        given.dequantize()
    with torch.no_grad():
        assert torch.equal(given.dequantize(), q.dequantize())
