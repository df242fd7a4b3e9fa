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


def test_dropped_elements_are_zero_whatever_they_held(tt):
    x = torch.full((1000,), np.inf, device="cuda")
    x[::3] = np.nan
    y = tt.dropout(x, 0.4, seed=3)
    keep = torch.from_numpy(half_words(1000, 3, 0) >= round(65536 * 0.4)).cuda()
    assert (y[~keep] == 0).all() and torch.equal(torch.isnan(y), keep & torch.isnan(x)) and (y[keep & ~torch.isnan(x)] == np.inf).all()
    assert (tt.dropout(x, 1.0, seed=3) == 0).all()


@pytest.mark.parametrize("layout", ["transposed", "sliced", "shifted", "expanded gradient", "scalar", "empty"])
def test_strides_and_shapes(tt, layout):
    x = torch.randn(40, 56, device="cuda")
    if layout == "transposed":
        x = x.t()
    elif layout == "sliced":
        x = x[::2, 3:50]
    elif layout == "shifted":
        x = torch.randn(40 * 56 + 1, device="cuda")[1:].view(40, 56)
    elif layout == "scalar":
        x = x[0, 0]
    elif layout == "empty":
        x = x[:0]
    a = x.detach().requires_grad_(True)
    y = tt.dropout(a, 0.3, seed=5, step=2)
    assert torch.equal(y.detach().cpu(), plain(x.cpu(), 0.3, 5, 2))
    (g,) = torch.autograd.grad(y.sum(), a)  # an expanded gradient
    assert torch.equal(g.cpu(), plain(torch.ones(x.shape), 0.3, 5, 2))


def test_gradient_of_the_gradient(tt):
    x = torch.randn(100, device="cuda", dtype=torch.float32, requires_grad=True)
    g = torch.randn(100, device="cuda", requires_grad=True)
    y = tt.dropout(x, 0.5, seed=9)
    (gx,) = torch.autograd.grad(y, x, g, create_graph=True)
    (gg,) = torch.autograd.grad(gx.square().sum(), g)
    mask = plain(torch.ones(100), 0.5, 9, 0).cuda()
    assert torch.equal(gg, 2 * g * mask * mask)


@pytest.mark.parametrize("kind", [torch.int32, torch.int64])
def test_step_on_the_device(tt, kind):
    """A captured forward and backward takes another mask when the step was changed, and the backward pass its own forward
    pass's mask even when the step has moved on."""
    x = torch.randn(500, device="cuda", requires_grad=True)
    g = torch.randn(500, device="cuda")
    step = torch.zeros(1, dtype=kind, device="cuda")
    y = tt.dropout(x, 0.5, seed=2, step=step)
    step += 1
    (gx,) = torch.autograd.grad(y, x, g)
    assert torch.equal(gx.cpu(), plain(g.cpu(), 0.5, 2, 0))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        z = x.detach().clone().requires_grad_(True)
        torch.autograd.grad(tt.dropout(z, 0.5, seed=2, step=step), z, g)
        with torch.cuda.graph(graph, stream=side):
            y = tt.dropout(z, 0.5, seed=2, step=step)
            step += 1
            (gz,) = torch.autograd.grad(y, z, g)
    torch.cuda.synchronize()
    for k in range(3):
        step.fill_(2**31 - 1 + k if kind == torch.int32 and k == 0 else 10 + k)
        torch.cuda.synchronize()
        now = int(step)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y.detach().cpu(), plain(z.detach().cpu(), 0.5, 2, now))
        assert torch.equal(gz.cpu(), plain(g.cpu(), 0.5, 2, now))


def test_more_than_2_to_the_32_elements(tt):
    n = 2**32 + 100
    x = torch.ones(n, dtype=torch.bfloat16, device="cuda")
    y = tt.dropout(x, 0.5, seed=77, step=1)
    for first in (0, 2**29 - 4, 2**29):  # groups of eight elements
        m = min(64, n - 8 * first)
        keep = half_words(m, 77, 1, first) >= 32768
        assert np.array_equal((y[8 * first : 8 * first + m] != 0).cpu().numpy(), keep)


def test_mean_is_kept(tt):
    """2^24 draws at p = 0.1: the mean of the kept ones within six standard deviations of 1."""
    n = 2**24
    y = tt.dropout(torch.ones(n, device="cuda"), 0.1, seed=4)
    p = round(6553.6) / 65536
    assert abs(float(y.double().mean()) - 1) < 6 * (p / (1 - p) / n) ** 0.5


def test_refusals(tt):
    x = torch.ones(8, device="cuda")
    for kw, match in [({"p": 1.5}, "between 0 and 1"), ({"p": float("nan")}, "between 0 and 1"), ({"seed": -1}, "seed"),
                      ({"seed": 2**64}, "seed"), ({"step": -1}, "step"), ({"step": 2**32}, "step"),
                      ({"step": torch.zeros(2, dtype=torch.int64, device="cuda")}, "step"),
                      ({"step": torch.zeros(1, device="cuda")}, "step"),
                      ({"step": torch.zeros(1, dtype=torch.int64)}, "CUDA")]:
        with pytest.raises(ValueError, match=match):
            tt.dropout(x, **({"p": 0.5, "seed": 1} | kw))
    with pytest.raises(ValueError, match="float32"):
        tt.dropout(x.int(), 0.5, seed=1)
    with pytest.raises(ValueError, match="CUDA"):
        tt.dropout(x.cpu(), 0.5, seed=1)


def test_gradient_against_differences(tt):
    """Dropout is linear: with p = 1/2 and whole numbers the difference along a direction is the gradient's product exactly."""
    g = torch.Generator(device="cuda").manual_seed(3)
    x = torch.randint(-9, 10, (300,), generator=g, device="cuda").float().requires_grad_(True)
    d, w = (torch.randint(-9, 10, (300,), generator=g, device="cuda").float() for _ in range(2))
    (grad,) = torch.autograd.grad(tt.dropout(x, 0.5, seed=8), x, w)
    up, down = (tt.dropout(x.detach() + s * d, 0.5, seed=8) for s in (1, -1))
    assert ((up - down) * w).sum() / 2 == (grad * d).sum()
