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
    few = T <= 128 or V <= 64  # g in two pieces: the rounding of the second one, 16 bits further down
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


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("rows,k,v", [(129, 8, 3), (515, 9, 2), (2000, 64, 64), (2000, 72, 65), (987, 20, 4), (21000, 40, 1),
                                      (40000, 33, 31), (3000, 2001, 33)])
def test_few_categories(tt, rows, k, v, dtype):
    """The differences of few categories cancel in the gradients of x: up to 64 are held in two pieces."""
    x, w, y, bias = batch(rows, k, v, DTYPES[dtype], rows + v)
    check(tt, x, w, y, bias, "mean" if rows % 2 else "none")


@pytest.mark.parametrize("which", ["x", "w", "bias"])
def test_one_gradient_of_few_categories(tt, which):
    """Each gradient by itself is that of all three; rows without a target keep theirs at zero."""
    x, w, y, bias = batch(700, 50, 11, torch.bfloat16, 12)
    leaves = {"x": x, "w": w, "bias": bias}

    def grads(names):
        t = {n: v.clone().requires_grad_(n in names) for n, v in leaves.items()}
        loss = tt.softmax_cross_entropy(t["x"], t["w"], y, bias=t["bias"])
        return dict(zip(names, torch.autograd.grad(loss, [t[n] for n in names])))

    all_three = grads(["x", "w", "bias"])
    assert torch.equal(grads([which])[which], all_three[which])
    assert torch.equal(all_three["x"][y == -100], torch.zeros_like(x[y == -100])) and bool((y == -100).any())


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


@pytest.mark.parametrize("dtype", list(DTYPES))
def test_categories_that_cannot_occur(tt, dtype):
    """A bias of -inf leaves a category out; a row without any category has loss inf and no gradient, a target that cannot
    occur loss inf and the gradient of the others."""
    x, w, y, bias = batch(60, 48, 300, DTYPES[dtype], 8, ignored=0)
    bias[torch.arange(0, 300, 3, device="cuda")] = -math.inf
    y = y // 3 * 3 + 1
    check(tt, x, w, y, bias, "none")
    y[7] = 9  # cannot occur
    loss = tt.softmax_cross_entropy(x, w, y, bias=bias, reduction="none")
    assert loss[7] == math.inf and torch.isfinite(loss[torch.arange(60, device="cuda") != 7]).all()
    b = torch.full_like(bias, -math.inf).requires_grad_(True)
    leaves = [t.clone().requires_grad_(True) for t in (x, w)]
    loss = tt.softmax_cross_entropy(*leaves, y, bias=b, reduction="sum")
    assert loss == math.inf
    loss.backward()
    for t in (*leaves, b):
        assert torch.equal(t.grad, torch.zeros_like(t))


def test_lowest_biases_count_as_any(tt):
    """The type's lowest value in place of -inf: categories of probability 0."""
    x, w, y, bias = batch(40, 32, 90, torch.bfloat16, 9, ignored=0)
    y = y % 30
    bias[30:] = torch.finfo(torch.float32).min
    check(tt, x, w, y, bias, "mean")
    few = tt.softmax_cross_entropy(x, w[:30].clone(), y, bias=bias[:30].clone(), reduction="none")
    assert torch.equal(few, tt.softmax_cross_entropy(x, w, y, bias=bias, reduction="none"))


@pytest.mark.parametrize("index", [-100, 0, 5, 2**40])
def test_rows_that_do_not_count(tt, index):
    x, w, y, bias = batch(130, 40, 66, torch.bfloat16, 10, ignored=0)
    y = torch.where(torch.arange(130, device="cuda") % 3 == 0, index, torch.where(y == index, 1, y))
    check(tt, x, w, y, bias, "mean", ignore=index)
    check(tt, x, w, torch.full_like(y, index), bias, "mean", ignore=index)  # a mean over no rows is 0
    check(tt, x, w, torch.full_like(y, index), bias, "none", ignore=index)


def test_targets_out_of_range_give_nan(tt):
    x, w, y, bias = batch(9, 16, 20, torch.bfloat16, 11, ignored=0)
    for bad in (20, -1, 2**40, -(2**62)):
        y[4] = bad
        leaf = x.clone().requires_grad_(True)
        loss = tt.softmax_cross_entropy(leaf, w, y, bias=bias, reduction="none")
        others = torch.arange(9, device="cuda") != 4
        assert torch.isnan(loss[4]) and torch.isfinite(loss[others]).all()
        assert torch.isnan(tt.softmax_cross_entropy(x, w, y, bias=bias))
        loss.sum().backward()
        assert torch.isnan(leaf.grad[4]).all() and torch.isfinite(leaf.grad[others]).all()
    tt.check_operator_errors()


def test_rows_that_are_not_finite(tt):
    """Infinities and NaN in a row of x are in its own loss and gradient alone (and in the weights' gradient)."""
    x, w, y, bias = batch(200, 24, 70, torch.bfloat16, 12, ignored=0)
    want = tt.softmax_cross_entropy(x, w, y, bias=bias, reduction="none")
    for bad in (math.inf, -math.inf, math.nan):
        z = x.clone()
        z[150, 3] = bad
        leaf = z.requires_grad_(True)
        loss = tt.softmax_cross_entropy(leaf, w, y, bias=bias, reduction="none")
        others = torch.arange(200, device="cuda") != 150
        assert torch.isnan(loss[150]) and torch.equal(loss[others], want[others])
        loss.sum().backward()
        assert torch.isnan(leaf.grad[150]).all() and torch.isfinite(leaf.grad[others]).all()


@pytest.mark.parametrize("layout", ["transposed", "sliced", "odd pitch", "expanded rows", "shifted", "three dimensions", "int32"])
def test_strides_and_shapes(tt, layout):
    x, w, y, bias = batch(72, 40, 130, torch.bfloat16, 13)
    want = [tt.softmax_cross_entropy(*(leaves := [t.clone().requires_grad_(True) for t in (x, w)]), y, bias=bias)]
    want += torch.autograd.grad(want[0], leaves)
    if layout == "transposed":
        a, b = x.t().contiguous().t(), w.t().contiguous().t()
    elif layout == "sliced":
        a, b = torch.empty(72, 88, dtype=x.dtype, device="cuda")[:, 8:48].copy_(x), torch.empty(260, 40, dtype=x.dtype, device="cuda")[::2].copy_(w)
    elif layout == "odd pitch":
        a, b = torch.empty(72, 41, dtype=x.dtype, device="cuda")[:, :40].copy_(x), torch.empty(130, 43, dtype=x.dtype, device="cuda")[:, :40].copy_(w)
    elif layout == "shifted":
        a = torch.empty(72 * 40 + 1, dtype=x.dtype, device="cuda")[1:].view(72, 40).copy_(x)
        b = torch.empty(130 * 40 + 3, dtype=x.dtype, device="cuda")[3:].view(130, 40).copy_(w)
    elif layout == "expanded rows":
        a, b = x[:1].expand(72, 40), w
        leaf = x[:1].repeat(72, 1).requires_grad_(True)
        want = [tt.softmax_cross_entropy(leaf, lw := w.clone().requires_grad_(True), y, bias=bias)]
        want += torch.autograd.grad(want[0], (leaf, lw))
    elif layout == "three dimensions":
        a, b, y = x.view(6, 12, 40), w, y.view(6, 12)
        want[1] = want[1].view(6, 12, 40)
    else:
        a, b, y = x, w, y.int()
    a, b = a.detach().requires_grad_(True), b.detach().requires_grad_(True)
    loss = tt.softmax_cross_entropy(a, b, y, bias=bias)
    got = [loss, *torch.autograd.grad(loss, (a, b))]
    for g, t in zip(got, want):
        assert torch.equal(g, t)
    each = tt.softmax_cross_entropy(a, b, y, bias=bias, reduction="none")
    assert each.shape == y.shape
    tt.check_operator_errors()


def test_only_some_gradients(tt):
    x, w, y, bias = batch(90, 40, 200, torch.bfloat16, 14)
    every = [t.clone().requires_grad_(True) for t in (x, w, bias)]
    want = torch.autograd.grad(tt.softmax_cross_entropy(every[0], every[1], y, bias=every[2]), every)
    for some in ([0], [1], [2], [0, 2], [1, 2]):
        t = [v.clone().requires_grad_(i in some) for i, v in enumerate((x, w, bias))]
        got = torch.autograd.grad(tt.softmax_cross_entropy(t[0], t[1], y, bias=t[2]), [t[i] for i in some])
        for g, i in zip(got, some):
            if i == 2 or some != [2]:
                assert torch.equal(g, want[i]) or i < 2, (some, i)
            if i < 2:  # other sums of logits where the bias' gradient is not asked for
                torch.testing.assert_close(g.double(), want[i].double(), rtol=2**-6, atol=float(want[i].abs().max()) * 2**-7)
    plain = tt.softmax_cross_entropy(x, w, y, bias=bias)
    assert not plain.requires_grad
    with torch.no_grad():
        assert not tt.softmax_cross_entropy(every[0], every[1], y, bias=every[2]).requires_grad


def test_no_rows(tt):
    w = torch.ones(5, 8, dtype=torch.bfloat16, device="cuda", requires_grad=True)
    x = torch.ones(0, 8, dtype=torch.bfloat16, device="cuda", requires_grad=True)
    y = torch.zeros(0, dtype=torch.int64, device="cuda")
    for reduction in ("mean", "sum"):
        loss = tt.softmax_cross_entropy(x, w, y, reduction=reduction)
        assert loss == 0 and loss.dtype == torch.float32
        gx, gw = torch.autograd.grad(loss, (x, w))
        assert gx.shape == (0, 8) and torch.equal(gw, torch.zeros_like(w))
    assert tt.softmax_cross_entropy(x, w, y, reduction="none").shape == (0,)


def test_what_autograd_refuses(tt):
    x, w, y, _ = batch(20, 16, 30, torch.bfloat16, 15, bias=False)
    a, b = x.clone().requires_grad_(True), w.clone().requires_grad_(True)
    loss = tt.softmax_cross_entropy(a, b, y)
    with pytest.raises(RuntimeError, match="second derivative"):
        torch.autograd.grad(loss, a, create_graph=True)
    loss = tt.softmax_cross_entropy(a, b, y)
    with torch.no_grad():
        b.add_(1.0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()
    import torch.autograd.forward_ad as fw

    with fw.dual_level():
        with pytest.raises((RuntimeError, NotImplementedError)):
            tt.softmax_cross_entropy(fw.make_dual(x, torch.ones_like(x)), w, y)
    with pytest.raises(RuntimeError):
        torch.func.vmap(lambda t: tt.softmax_cross_entropy(t, w, y))(torch.stack([x, x]))


def test_captured_steps_replay_on_new_inputs(tt):
    """Two graphs of forward and backward share their inputs, run in turn beside eager calls, and give what eager calls do;
    an eager graph of the same leaves (of the same stream, as torch wants it) lives while they are captured."""
    x, w, y, bias = batch(140, 72, 900, torch.bfloat16, 16)
    leaves = [t.clone().requires_grad_(True) for t in (x, w, bias)]

    def run(reduction):
        loss = tt.softmax_cross_entropy(leaves[0], leaves[1], y, bias=leaves[2], reduction=reduction)
        return loss.detach(), *torch.autograd.grad(loss, leaves)

    graphs = []
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        alive = tt.softmax_cross_entropy(leaves[0], leaves[1], y, bias=leaves[2])
        for reduction in ("mean", "sum"):
            run(reduction)
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=side):
                out = run(reduction)
            graphs.append((reduction, graph, out))
        kept = torch.autograd.grad(alive, leaves)
    torch.cuda.synchronize()
    for seed in range(3):
        x2, w2, y2, b2 = batch(140, 72, 900, torch.bfloat16, 50 + seed)
        with torch.no_grad():
            for t, v in zip((*leaves, y), (x2, w2, b2, y2)):
                t.copy_(v)
        torch.cuda.synchronize()
        for reduction, graph, out in graphs:
            graph.replay()
            eager = run(reduction)
            torch.cuda.synchronize()
            for a, b in zip(out, eager):
                assert torch.equal(a, b)
    assert all(torch.isfinite(t).all() for t in kept)
    tt.check_operator_errors()


def test_backward_into_leaves_captured_beside_an_eager_graph(tt):
    """loss.backward() of a captured step, with an eager graph of the same leaves alive."""
    x, w, y, _ = batch(30, 32, 50, torch.bfloat16, 17, bias=False)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        a, b = x.clone().requires_grad_(True), w.clone().requires_grad_(True)
        tt.softmax_cross_entropy(a, b, y).backward()
        want = a.grad.clone(), b.grad.clone()
        alive = tt.softmax_cross_entropy(a, b, y)
        a.grad = b.grad = None
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            tt.softmax_cross_entropy(a, b, y).backward()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(a.grad, want[0]) and torch.equal(b.grad, want[1])
        assert torch.isfinite(alive)


def test_another_stream_and_threads(tt):
    import threading

    x, w, y, bias = batch(300, 64, 2000, torch.bfloat16, 18)
    want = tt.softmax_cross_entropy(x, w, y, bias=bias)
    torch.cuda.synchronize()
    got = {}

    def work(i):
        s = torch.cuda.Stream()
        with torch.cuda.stream(s):
            a, b = x.clone().requires_grad_(True), w.clone().requires_grad_(True)
            for _ in range(5):
                loss = tt.softmax_cross_entropy(a, b, y, bias=bias)
                grads = torch.autograd.grad(loss, (a, b))
            s.synchronize()
            got[i] = (loss, *grads)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for i in range(4):
        assert torch.equal(got[i][0], want)
        for a, b in zip(got[i], got[0]):
            assert torch.equal(a, b)


def test_weights_of_more_than_2_to_the_31_elements(tt):
    V, K = 16_000_000, 136
    g = torch.Generator(device="cuda").manual_seed(1)
    w = torch.empty(V, K, dtype=torch.bfloat16, device="cuda")
    for at in range(0, V, 1_000_000):
        w[at : at + 1_000_000] = torch.randn(1_000_000, K, generator=g, device="cuda") * 0.1
    x = torch.randn(3, K, generator=g, device="cuda").bfloat16()
    y = torch.tensor([5, V - 1, V - 70_000], device="cuda")
    loss = tt.softmax_cross_entropy(x, w, y, reduction="none")
    logits = torch.cat([x.double() @ w[at : at + 1_000_000].double().t() for at in range(0, V, 1_000_000)], 1)
    want = torch.logsumexp(logits, 1) - logits.gather(1, y[:, None])[:, 0]
    # as in expected(): a logit's sum, and the normaliser's exponentials and additions (at most V / 4096 per partial sum)
    tol = 4e-6 * (1 + want.abs()) + (V / 4096 + 200) * 2.0**-24
    assert ((loss.double() - want).abs() <= tol).all()
    leaf = w.requires_grad_(True)
    (dw,) = torch.autograd.grad(tt.softmax_cross_entropy(x, leaf, y, reduction="sum"), leaf)
    for at in (5, V - 1, V - 70_000, V // 2):
        p = torch.exp(logits[:, at] - torch.logsumexp(logits, 1)) - (y == at).double()
        exact = p @ x.double()
        assert ((dw[at].double() - exact).abs() <= 2.0**-7 * exact.abs() + 1e-4 * exact.abs().max()).all()
    tt.check_operator_errors()


def test_weights_of_rows_that_are_nan(tt):
    """NaN among the weights of 'none': the row's own gradient and the weights' are NaN, the other rows' are not; also where
    it stands alone."""
    x, w, y, _ = batch(10, 16, 40, torch.bfloat16, 19, bias=False, ignored=0)
    for others in (1.0, 0.0):
        a, b = x.clone().requires_grad_(True), w.clone().requires_grad_(True)
        weight = torch.full((10,), others, device="cuda")
        weight[3] = math.nan
        tt.softmax_cross_entropy(a, b, y, reduction="none").backward(weight)
        rest = torch.arange(10, device="cuda") != 3
        assert torch.isnan(a.grad[3]).all() and torch.isfinite(a.grad[rest]).all() and torch.isnan(b.grad).all()


@pytest.mark.parametrize("which", [0, 1, 2])
def test_gradients_against_differences(tt, which):
    """Central differences of the loss along a direction.  x and w are multiples of 2^-6 below 2, so that x +- d and w +- d are
    exact in bfloat16.  The difference's own error: a third of a derivative, at most R^3 / 6 with R the range of the logits'
    change; the losses' (1e-6 each); the gradient's: 2^-8 of each element, twice (g and the result)."""
    g = torch.Generator(device="cuda").manual_seed(23)

    def grid(*shape):
        return (torch.randint(-64, 65, shape, generator=g, device="cuda") / 64.0)

    x, w, bias = grid(150, 48), grid(200, 48) / 4, torch.randn(200, generator=g, device="cuda")
    w = torch.round(w * 64) / 64
    y = torch.randint(0, 200, (150,), generator=g, device="cuda")
    values = [x, w, bias]
    d = torch.where(torch.rand(values[which].shape, generator=g, device="cuda") < 0.5, -1.0, 1.0) / 64

    def loss(sign):
        v = [t + sign * d if i == which else t for i, t in enumerate(values)]
        assert torch.equal(v[0].bfloat16().float(), v[0]) and torch.equal(v[1].bfloat16().float(), v[1])
        return tt.softmax_cross_entropy(v[0].bfloat16(), v[1].bfloat16(), y, bias=v[2]).double()

    leaves = [x.bfloat16(), w.bfloat16(), bias.clone()]
    leaf = leaves[which].requires_grad_(True)
    (grad,) = torch.autograd.grad(tt.softmax_cross_entropy(leaves[0], leaves[1], y, bias=leaves[2]), leaf)
    slope = (grad.double() * d.double()).sum()
    change = d.double() @ w.double().t() if which == 0 else (x.double() @ d.double().t() if which == 1 else d.double()[None])
    reach = float((change.amax(1) - change.amin(1)).max())
    size = float((grad.double().abs() * d.double().abs()).sum())
    assert abs(float(loss(1) - loss(-1)) / 2 - float(slope)) <= reach**3 / 6 + 1e-6 * 6 + 2 * 2.0**-8 * size
    assert abs(float(slope)) > 1e-4
