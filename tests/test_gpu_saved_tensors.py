"""Gradients under hooks on saved tensors: what the forward pass saved may come back with other strides."""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def tt():
    import tt_thrml_b200

    return tt_thrml_b200


def values(rows, k, v, seed):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, k, generator=g).bfloat16().cuda()
    w = (torch.randn(v, k, generator=g) / math.sqrt(k)).bfloat16().cuda()
    y = torch.randint(0, v, (rows,), generator=g)
    y = torch.where(torch.rand(rows, generator=g) < 0.1, -100, y).cuda()
    return x, w, y, torch.randn(v, generator=g).cuda()


def padded(t, pitch, first=0):
    out = torch.zeros(t.shape[0] * pitch + first, dtype=t.dtype, device=t.device)
    return out[first:].view(t.shape[0], pitch)[:, : t.shape[1]].copy_(t)


def transposed(t):
    return t.t().contiguous().t()


# how x and w lie: read as they lie, or laid out again; a dense copy of them changes that for one, the other, both or neither
LAYOUTS = {
    "x as it lies, w odd": (1001, lambda x: padded(x, 1008), lambda w: w),
    "x odd, w as it lies": (1001, lambda x: x, lambda w: padded(w, 1008)),
    "x odd pitch, w transposed": (40, lambda x: padded(x, 41), transposed),
    "x shifted, w transposed": (72, lambda x: padded(x, 72, 1), transposed),
    "both as they lie": (1001, lambda x: padded(x, 1008), lambda w: padded(w, 1016)),
    "both odd": (33, lambda x: x, lambda w: w),
    "both dense": (64, lambda x: x, lambda w: w),
}


def gradients(tt, x, w, y, bias, reduction="mean"):
    leaves = [t.detach().requires_grad_(True) for t in (x, w, bias)]
    loss = tt.softmax_cross_entropy(leaves[0], leaves[1], y, bias=leaves[2], reduction=reduction)
    return loss, leaves


@pytest.mark.parametrize("pinned", [False, True])
@pytest.mark.parametrize("reduction", ["mean", "none"])
@pytest.mark.parametrize("layout", list(LAYOUTS))
def test_saved_on_the_host(tt, layout, reduction, pinned):
    k, of_x, of_w = LAYOUTS[layout]
    x, w, y, bias = values(150, k, 333, k)
    a, b = of_x(x), of_w(w)
    assert torch.equal(a, x) and torch.equal(b, w)
    grad = torch.linspace(-1, 2, 150, device="cuda") if reduction == "none" else None
    loss, leaves = gradients(tt, x, w, y, bias, reduction)
    want = torch.autograd.grad(loss, leaves, grad)
    with torch.autograd.graph.save_on_cpu(pin_memory=pinned):
        loss, leaves = gradients(tt, a, b, y, bias, reduction)
        got = torch.autograd.grad(loss, leaves, grad)
    for g, t in zip(got, want):
        assert torch.equal(g, t)
    tt.check_operator_errors()


@pytest.mark.parametrize("k", [33, 64])
def test_saved_tensors_that_come_back_with_any_strides(tt, k):
    """Every saved tensor comes back with its last dimension strided and one element behind an aligned address."""
    x, w, y, bias = values(70, k, 90, 5)
    loss, leaves = gradients(tt, x, w, y, bias)
    want = torch.autograd.grad(loss, leaves)

    def strided(t):
        if not t.dim():
            return t.clone()
        out = torch.zeros((*t.shape, 2), dtype=t.dtype, device=t.device)[..., 1]
        return out.copy_(t)

    with torch.autograd.graph.saved_tensors_hooks(lambda t: t, strided):
        loss, leaves = gradients(tt, x, w, y, bias)
        got = torch.autograd.grad(loss, leaves)
    for g, t in zip(got, want):
        assert torch.equal(g, t)
    tt.check_operator_errors()


@pytest.mark.parametrize("change", [lambda t: t.cpu(), lambda t: t.double(),
                                    lambda t: t[:-1] if t.dtype == torch.bfloat16 or t.shape == (1,) else t],
                         ids=["device", "type", "size"])
def test_saved_tensors_that_are_others_are_refused(tt, change):
    x, w, y, bias = values(20, 24, 30, 6)
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t, change):
        loss, leaves = gradients(tt, x, w, y, bias)
        with pytest.raises(RuntimeError, match="saved tensor"):
            torch.autograd.grad(loss, leaves)
        step = torch.zeros(1, dtype=torch.int64, device="cuda")
        leaf = torch.ones(20, device="cuda", requires_grad=True)
        kept = tt.dropout(leaf, 0.5, seed=1, step=step)
        with pytest.raises(RuntimeError, match="saved tensor"):
            torch.autograd.grad(kept.sum(), leaf)


def test_dropout_saved_on_the_host(tt):
    x, g = torch.randn(500, device="cuda", requires_grad=True), torch.randn(500, device="cuda")
    step = torch.full((1,), 3, dtype=torch.int64, device="cuda")
    (want,) = torch.autograd.grad(tt.dropout(x, 0.5, seed=2, step=3), x, g)
    with torch.autograd.graph.save_on_cpu():
        y = tt.dropout(x, 0.5, seed=2, step=step)
        step += 1
        (got,) = torch.autograd.grad(y, x, g)
    assert torch.equal(got, want)


def test_a_readout_in_any_layout(tt):
    """A step of the readout (its own forward and backward pass in one call) on rows that are laid out again."""
    x, _, y, _ = values(150, 33, 70, 9)
    losses = []
    for units in (x, padded(x, 40), transposed(x)):
        r = tt.CategoricalReadout(33, 70, seed=4)
        losses.append((r.step(units, y), r.gradient[0].clone(), r.weights.clone()))
    for other in losses[1:]:
        assert all(torch.equal(a, b) for a, b in zip(losses[0], other))
