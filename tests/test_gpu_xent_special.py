"""Numbers that are not finite, or not far from that, in the cross entropy's inputs."""

import math

import pytest
import torch

from test_gpu_xent import DTYPES, batch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def tt():
    import tt_thrml_b200

    return tt_thrml_b200


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("rows,v", [(10, 40), (10, 300), (300, 40), (300, 700)])
@pytest.mark.parametrize("weight", [math.inf, -math.inf, math.nan])
def test_weights_of_rows_that_are_not_finite(tt, weight, rows, v, dtype):
    """They are in the row's own gradient (and in the weights'); the other rows' are what they are without that row's."""
    x, w, y, _ = batch(rows, 24, v, DTYPES[dtype], 19, bias=False, ignored=0)
    y[5] = -100
    weights = torch.linspace(0.5, 2.0, rows, device="cuda")

    def gradients():
        leaves = [t.clone().requires_grad_(True) for t in (x, w)]
        tt.softmax_cross_entropy(*leaves, y, reduction="none").backward(weights)
        return [t.grad for t in leaves]

    weights[3] = 0.0
    want, _ = gradients()
    weights[3] = weight
    got, dw = gradients()
    rest = torch.arange(rows, device="cuda") != 3
    assert torch.equal(got[rest], want[rest])
    assert not torch.isfinite(got[3]).any() and not torch.isfinite(dw).any()
    weights[3], weights[5] = 0.0, weight  # a row that does not count: its weight is in nothing
    got, dw = gradients()
    assert torch.equal(got, want) and torch.isfinite(dw).all()
