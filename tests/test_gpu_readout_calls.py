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
