"""Calls of the operators around dense programs that their documentation allows beside the ordinary ones."""

import pytest
import torch

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16


@pytest.fixture(scope="module")
def tt():
    import tt_thrml_b200

    return tt_thrml_b200


@pytest.fixture
def default_dtype():
    was = torch.get_default_dtype()
    yield torch.set_default_dtype
    torch.set_default_dtype(was)


@pytest.mark.parametrize("kind", [BF16, torch.float16, torch.float64])
def test_coded_moments_under_another_default_dtype(tt, default_dtype, kind):
    """The kernel reads and writes float32 scales, whatever type new tensors have by default."""
    g = torch.randn(3000, generator=torch.Generator().manual_seed(1), dtype=F32).cuda()

    def run():
        p = torch.zeros(3000, dtype=F32, device="cuda")
        opt = tt.AdamW([p], state_bits=8, seed=2)
        assert opt.exp_avg_scale.dtype == F32 and opt.exp_avg_sq_scale.dtype == F32
        for _ in range(3):
            opt.step([g])
        return [p, *(v for k, v in opt.state_dict().items() if k != "step")]

    want = run()
    default_dtype(kind)
    for a, b in zip(run(), want):
        assert a.dtype == b.dtype and torch.equal(a, b)
