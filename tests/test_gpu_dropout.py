"""Dropout on the GPU against the generator in 64-bit host arithmetic."""

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}


@pytest.fixture(scope="module")
def tt():
    import tt_thrml_b200

    return tt_thrml_b200


def half_words(n, seed, step, first=0):
    """The n 16-bit numbers that decide elements 8 * first and following."""
    g = np.arange(first, first + (n + 7) // 8, dtype=np.uint64)
    low, c32 = np.uint64(0xFFFFFFFF), np.uint64(32)
    c = [g & low, g >> c32, np.full_like(g, step & 0xFFFFFFFF), np.full_like(g, 0x44524F50)]
    k = [seed & 0xFFFFFFFF, seed >> 32]
    for _ in range(10):
        a, b = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        c = [(b >> c32) ^ c[1] ^ np.uint64(k[0]), b & low, (a >> c32) ^ c[3] ^ np.uint64(k[1]), a & low]
        k = [(k[0] + 0x9E3779B9) & 0xFFFFFFFF, (k[1] + 0xBB67AE85) & 0xFFFFFFFF]
    return np.stack([h for w in c for h in (w & np.uint64(0xFFFF), w >> np.uint64(16))], 1).reshape(-1)[:n].astype(np.int64)


def plain(x, p, seed, step):
    cut = round(65536 * p)
    keep = torch.from_numpy(half_words(x.numel(), seed, step) >= cut).view(x.shape)
    scale = torch.tensor(0.0 if cut == 65536 else 65536.0 / (65536.0 - cut), dtype=torch.float32)
    return torch.where(keep, (x.float() * scale), 0.0).to(x.dtype)


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("shape", [(1,), (7,), (8,), (3, 5), (64, 512), (1000, 33), (2, 3, 4, 5), (70001,)])
@pytest.mark.parametrize("p", [0.0, 0.1, 0.5, 1.0])
def test_values_and_gradients(tt, shape, dtype, p):
    x = torch.randn(shape, generator=torch.Generator().manual_seed(len(shape))).to(DTYPES[dtype])
    g = torch.randn(shape, generator=torch.Generator().manual_seed(9)).to(DTYPES[dtype])
    seed, step = 0xFEDCBA9876543210, 7
    a = x.cuda().requires_grad_(True)
    y = tt.dropout(a, p, seed=seed, step=step)
    assert torch.equal(y.detach().cpu(), plain(x, p, seed, step))
    y.backward(g.cuda())
    assert torch.equal(a.grad.cpu(), plain(g, p, seed, step))
