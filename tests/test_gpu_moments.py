"""Pair moments on the GPU against sums in 64 bits."""

import pytest
import torch

from tt_thrml_b200 import _native as nat

pytestmark = pytest.mark.gpu

BF16, F16 = torch.bfloat16, torch.float16


@pytest.fixture(scope="module")
def tt():
    import tt_thrml_b200

    return tt_thrml_b200


def rand(shape, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(shape, generator=g).to(dtype)


def ints(shape, top, seed):
    g = torch.Generator().manual_seed(seed)
    return torch.randint(-top, top + 1, shape, generator=g).float()


def exact(xs, ys, scales):
    """The 64-bit sums and the sum of the magnitudes of all terms."""
    w = sum(s * (x.double().t() @ y.double()) for x, y, s in zip(xs, ys, scales))
    a = sum(abs(s) * (x.double().abs().t() @ y.double().abs()) for x, y, s in zip(xs, ys, scales))
    return w, a, sum(s * x.double().sum(0) for x, s in zip(xs, scales)), sum(s * y.double().sum(0) for y, s in zip(ys, scales))


def bound(a, chains):
    """Products of 16-bit values are exact in float32.  One MMA adds 16 of them to the accumulator, each operand aligned
    to the largest within one float32 step (2^-23) of the sum of magnitudes: 17 steps per MMA, at most 64 MMAs before the
    sum moves to a register; there each of the chunks' additions rounds once, and the splits' ones once more."""
    mmas = min(64, -(-max(chains) // 16))
    adds = sum(-(-c // 1024) for c in chains) + 16
    return a * 2.0**-23 * (17 * mmas + adds)


SHAPES = [(1, 1, [1]), (1, 9, [3, 0]), (8, 64, [16, 16]), (65, 63, [17, 64]), (127, 129, [65, 1]), (128, 256, [512]),
          (129, 257, [513, 100]), (200, 1000, [1023, 2050]), (640, 72, [64, 128, 192]), (1000, 513, [4000, 70]),
          (64, 3, [5, 6, 7, 8, 9, 10]), (2, 300, [9000]), (2100, 2333, [70, 1100]), (2600, 2049, [129]), (1501, 3001, [1100, 1300])]


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("m,n,chains", SHAPES)
def test_moments_match_the_64_bit_sums(tt, m, n, chains, dtype):
    xs = [rand((c, m), dtype, 10 + i) for i, c in enumerate(chains)]
    ys = [rand((c, n), dtype, 50 + i) for i, c in enumerate(chains)]
    scales = [(-1.0) ** i / max(1, c) for i, c in enumerate(chains)]
    out, sx, sy = tt.pair_moments([x.cuda() for x in xs], [y.cuda() for y in ys], scales, units=True)
    w, a, wx, wy = exact(xs, ys, scales)
    assert ((out.cpu().double() - w).abs() <= bound(a, chains) + 1e-38).all()
    for got, want, ts in ((sx, wx, xs), (sy, wy, ys)):
        # 16 lanes or more, each at most ceil(chains / 16) additions, then 20 at most to join them, one per phase and its scale
        mags = sum(abs(s) * t.double().abs().sum(0) for t, s in zip(ts, scales))
        adds = sum(-(-c // 16) for c in chains) + 20 + 2 * len(chains)
        assert ((got.cpu().double() - want).abs() <= mags * adds * 2.0**-24 + 1e-38).all()
    again = tt.pair_moments([x.cuda() for x in xs], [y.cuda() for y in ys], scales)
    assert torch.equal(again, out)  # the same every time
    tt.check_operator_errors()


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("m,n,chains", [(300, 520, [3000, 700]), (130, 70, [100, 1]), (1, 1, [5000, 5000]), (2305, 2049, [300, 1100]), (1500, 2990, [1500, 1100])])
def test_whole_numbers_are_exact(tt, m, n, chains, dtype):
    xs = [ints((c, m), 8, i).to(dtype) for i, c in enumerate(chains)]
    ys = [(ints((c, n), 8, 20 + i) * 2 + 1).sign().to(dtype) for i, c in enumerate(chains)]
    out, sx, sy = tt.pair_moments([x.cuda() for x in xs], [y.cuda() for y in ys], [1.0, -2.0], units=True)
    w, _, wx, wy = exact(xs, ys, [1.0, -2.0])
    assert torch.equal(out.cpu().double(), w) and torch.equal(sx.cpu().double(), wx) and torch.equal(sy.cpu().double(), wy)


def test_accumulate_output_strides_and_untouched_columns(tt):
    x, y = ints((70, 90), 5, 1).to(BF16), ints((70, 130), 5, 2).to(BF16)
    w, _, wx, wy = exact([x], [y], [1.0])
    big = torch.full((90, 150), 3.0, device="cuda")
    sx, sy = torch.full((90,), 1.0, device="cuda"), torch.full((130,), 2.0, device="cuda")
    view = big[:, 7:137]
    for k in (1, 2):
        got = tt.pair_moments(x.cuda(), y.cuda(), out=(view, sx, sy), accumulate=True, units=True)
        assert got[0] is view
        assert torch.equal(view.cpu().double(), 3.0 + k * w)
        assert torch.equal(sx.cpu().double(), 1.0 + k * wx) and torch.equal(sy.cpu().double(), 2.0 + k * wy)
    tt.pair_moments(x.cuda(), y.cuda(), out=view)
    assert torch.equal(view.cpu().double(), w)
    assert (big[:, :7] == 3).all() and (big[:, 137:] == 3).all()


@pytest.mark.parametrize("m,n,pitch", [(2305, 2080, 2080), (2305, 2077, 2080), (2300, 2049, 2049), (2049, 2336, 2343),
                                       (2900, 4160, 4160), (2900, 4101, 4104), (2817, 4097, 4097)])
def test_sums_added_to_large_outputs(tt, m, n, pitch):
    """Whole numbers: rows that start on 16 bytes and others, tiles cut off in rows and columns."""
    x, y = ints((70, m), 5, 1).to(BF16), ints((70, n), 5, 2).to(BF16)
    w, _, _, _ = exact([x], [y], [1.0])
    start = ints((m, pitch), 9, 3)
    out = start.cuda()
    tt.pair_moments(x.cuda(), y.cuda(), 2.0, out=out[:, :n], accumulate=True)
    assert torch.equal(out[:, :n].cpu().double(), start[:, :n].double() + 2 * w)
    assert torch.equal(out[:, n:].cpu(), start[:, n:])
    tt.pair_moments(x.cuda(), y.cuda(), out=out[:, :n])
    assert torch.equal(out[:, :n].cpu().double(), w) and torch.equal(out[:, n:].cpu(), start[:, n:])


def test_strides_of_the_operands(tt):
    base = ints((400, 333), 6, 3).to(F16)
    y = ints((200, 48), 6, 4).to(F16)
    d = base.cuda()
    for cut in (lambda t: t[:200, 1:100], lambda t: t[::2, :64], lambda t: t.t()[:200, :399], lambda t: t[:1, :40].expand(200, 40),
                lambda t: t[100:300, 8:80:3]):
        x = cut(base)
        out, sx, _ = tt.pair_moments(cut(d), y.cuda(), units=True)
        w, _, wx, _ = exact([x], [y], [1.0])
        assert torch.equal(out.cpu().double(), w) and torch.equal(sx.cpu().double(), wx)


def test_no_chains_give_zeros_or_leave_the_sum(tt):
    x, y = torch.empty((0, 20), dtype=BF16, device="cuda"), torch.empty((0, 33), dtype=BF16, device="cuda")
    out, sx, sy = tt.pair_moments(x, y, units=True)
    assert not out.any() and not sx.any() and not sy.any()
    out.fill_(4.0)
    tt.pair_moments([x, x], [y, y], [1.0, 2.0], out=out, accumulate=True)
    assert (out == 4).all()


def test_values_that_are_not_finite_stay_with_their_units(tt):
    x, y = torch.ones((130, 70), dtype=BF16), torch.ones((130, 300), dtype=BF16)
    x[64, 3] = float("nan")
    y[129, 299] = float("inf")
    out, sx, sy = (t.cpu() for t in tt.pair_moments(x.cuda(), y.cuda(), units=True))
    bad = torch.zeros_like(out, dtype=torch.bool)
    bad[3] = True
    bad[:, 299] = True
    assert torch.equal(~torch.isfinite(out), bad) and (out[~bad] == 130).all()
    assert torch.isnan(sx[3]) and torch.isinf(sy[299]) and torch.isfinite(sx[4:]).all() and torch.isfinite(sy[:299]).all()


def test_a_phase_of_scale_zero_is_zero_times_its_sums(tt):
    x, y = torch.ones((70, 40), dtype=BF16), torch.ones((70, 90), dtype=BF16)
    z, w = x.clone(), y.clone()
    z[5, 7] = float("nan")
    w[69, 80] = float("inf")
    out, sx, sy = (t.cpu() for t in tt.pair_moments([x.cuda(), z.cuda()], [y.cuda(), w.cuda()], [1.0, 0.0], units=True))
    bad = torch.zeros_like(out, dtype=torch.bool)
    bad[7] = True
    bad[:, 80] = True
    assert torch.equal(torch.isnan(out), bad) and (out[~bad] == 70).all()
    assert torch.equal(torch.isnan(sx), bad[:, 0]) and torch.equal(torch.isnan(sy), bad[0])
    assert (sx[~bad[:, 0]] == 70).all() and (sy[~bad[0]] == 70).all()


def test_gradient_of_the_log_likelihood_by_differences(tt):
    """d log p / d W of a small Boltzmann machine of two spin blocks, by enumeration, against the moments of its own
    distribution given as weighted phases: data minus model, and against differences of the log likelihood."""
    V, H = 3, 2
    g = torch.Generator().manual_seed(0)
    W = torch.randn((V, H), generator=g).double()
    states = torch.tensor([[1.0 if k >> i & 1 else -1.0 for i in range(V + H)] for k in range(2 ** (V + H))], dtype=torch.float64)
    v, h = states[:, :V], states[:, V:]
    data = torch.tensor([[1.0, -1.0, 1.0], [-1.0, -1.0, 1.0]], dtype=torch.float64)

    def log_likelihood(W):
        def free(v):  # log sum over h of exp(v W h)
            hs = torch.tensor([[a, b] for a in (-1.0, 1.0) for b in (-1.0, 1.0)], dtype=torch.float64)
            return torch.logsumexp((v @ W) @ hs.t(), 1)

        vs = torch.tensor([[1.0 if k >> i & 1 else -1.0 for i in range(V)] for k in range(2**V)], dtype=torch.float64)
        return (free(data) - torch.logsumexp(free(vs), 0)).mean()

    # model phase: every state with its probability; data phase: v with the mean of h given v, split into states
    logp = ((v @ W) * h).sum(1)
    p = torch.softmax(logp, 0)
    hs = torch.tensor([[a, b] for a in (-1.0, 1.0) for b in (-1.0, 1.0)], dtype=torch.float64)
    grad = torch.zeros((V, H), dtype=torch.float32, device="cuda")
    for k in range(len(p)):  # one chain per phase, weighted
        grad = tt.pair_moments(v[k : k + 1].to(BF16).cuda(), h[k : k + 1].to(BF16).cuda(), -p[k].item(), out=grad, accumulate=True)
    for d in data:
        q = torch.softmax(hs @ (d @ W), 0)
        for k in range(4):
            grad = tt.pair_moments(d[None].to(BF16).cuda(), hs[k : k + 1].to(BF16).cuda(), q[k].item() / 2, out=grad, accumulate=True)
    eps = 1e-5
    for i in range(V):
        for j in range(H):
            up, down = W.clone(), W.clone()
            up[i, j] += eps
            down[i, j] -= eps
            diff = (log_likelihood(up) - log_likelihood(down)) / (2 * eps)
            # 40 float32 additions of terms that sum to at most 2, each weight rounded once
            assert abs(grad[i, j].item() - diff.item()) < 2 * 41 * 2.0**-24 + 1e-9


def test_two_captured_graphs_on_two_streams(tt):
    xs, ys = [ints((300, 140), 5, i).to(BF16) for i in (1, 2)], [ints((300, 270), 5, i).to(BF16) for i in (3, 4)]
    held = [(x.cuda(), y.cuda()) for x, y in zip(xs, ys)]
    tt.pair_moments(*held[0])
    graphs, outs = [], []
    for x, y in held:
        g = torch.cuda.CUDAGraph()
        with nat.capturing(g):
            outs.append(tt.pair_moments(x, y, 0.5, units=True))
        graphs.append(g)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in graphs]
    for _ in range(10):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    for x, y, o in zip(xs, ys, outs):
        w, _, wx, wy = exact([x], [y], [0.5])
        assert torch.equal(o[0].cpu().double(), w) and torch.equal(o[1].cpu().double(), wx) and torch.equal(o[2].cpu().double(), wy)


def test_refusals(tt):
    x, y = torch.ones((4, 5), dtype=BF16, device="cuda"), torch.ones((4, 6), dtype=BF16, device="cuda")
    buffer = torch.zeros((8, 64), dtype=torch.uint8, device="cuda")
    for args, kw, exc in [
        ((x.float(), y.float()), {}, ValueError),
        ((x, y.half()), {}, ValueError),
        ((x.cpu(), y.cpu()), {}, ValueError),
        ((x, y[:3]), {}, ValueError),
        (([x, x], [y]), {}, ValueError),
        (([x, x[:, :4]], [y, y], [1, 1]), {}, ValueError),
        (([x] * 7, [y] * 7), {}, ValueError),
        (([x, x], [y, y], [1.0]), {}, ValueError),
        ((x[:, :0], y), {}, ValueError),
        ((x, y), {"accumulate": True}, ValueError),
        ((x, y), {"out": torch.empty((6, 5), device="cuda")}, ValueError),
        ((x, y), {"out": torch.empty((6, 5), device="cuda").t()}, ValueError),
        ((x, y), {"out": torch.empty((5, 6), device="cuda").half()}, ValueError),
        ((x, y), {"out": (torch.empty((5, 6), device="cuda"), torch.empty(4, device="cuda"), torch.empty(6, device="cuda")),
                  "units": True}, ValueError),
        ((buffer.view(BF16)[:4, :5], y), {"out": buffer.view(torch.float32)[:5, :6]}, ValueError),
        ((x.clone().requires_grad_(True), y), {}, RuntimeError),
    ]:
        with pytest.raises(exc):
            tt.pair_moments(*args, **kw)
