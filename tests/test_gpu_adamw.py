"""AdamW on the GPU against plain implementations in 64 bits (float32 moments) and bit for bit (8-bit codes)."""

import math

import numpy as np
import pytest
import torch

from tt_thrml_b200 import _native as nat

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
U = 2.0**-24
HYPER = dict(lr=3e-3, betas=(0.9, 0.99), eps=1e-8, weight_decay=0.1)


@pytest.fixture(scope="module")
def tt():
    import tt_thrml_b200

    return tt_thrml_b200


def rand(shape, dtype, seed, std=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * std).to(dtype)


def formula64(p, g, m, v, t, h, dtype, roundings=7.1):
    """One step in 64 bits from the given values, with the bounds that the float32 roundings leave.  `roundings` of
    the update itself: 7 correctly rounded operations, or 13 with the hardware's square root (two steps of 2^-23 at
    most) and quotient (two likewise)."""
    p, g, m, v = (x.double() for x in (p, g, m, v))
    (b1, b2), lr, wd, eps = h["betas"], h["lr"], h["weight_decay"], h["eps"]
    m1, v1 = b1 * m + (1 - b1) * g, b2 * v + (1 - b2) * g * g
    step, r = lr / (1 - b1**t), 1 / math.sqrt(1 - b2**t)
    denom = v1.sqrt() * r + eps
    upd = step * m1 / denom
    p1 = p * (1 - lr * wd) - upd
    # a product with a rounded coefficient: two roundings; g^2 one more; the sum one
    em = U * (2.01 * (b1 * m.abs() + (1 - b1) * g.abs()) + m1.abs())
    ev = U * (2.01 * b2 * v + 3.02 * (1 - b2) * g * g + v1) + 1.0e-44
    # the update: m's bound; v's through the square root (half of it, relative); the root, its coefficient, the product
    # and the sum of the denominator, the quotient, the rounded step size and its product: seven roundings
    # (the quantity v / 2 v1 bounds sqrt's change; where v1 is 0, m1 is 0 too or g is 0 and nothing changes)
    rel_v = torch.where(v1 > 0, ev / (2 * v1.clamp_min(1e-300)), torch.zeros_like(v1))
    eu = step * em / denom + upd.abs() * (roundings * U + rel_v)
    ep = 2.01 * U * p.abs() + eu + U * p1.abs()
    if dtype != F32:
        ep = ep + torch.finfo(dtype).eps / 2 * (p1.abs() + ep) + torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
    return (p1, m1, v1), (ep, em, ev)


SIZES = [(1,), (255,), (256,), (257,), (2048,), (2049,), (5, 333), (64, 130), (0,), (70000,), (3, 1, 5, 7)]
TYPES = [(F32, F32), (BF16, BF16), (BF16, F32), (F16, F16), (F16, F32)]


@pytest.mark.parametrize("count", [1, 11, 60])
@pytest.mark.parametrize("ptype,gtype", TYPES)
def test_steps_match_the_formula(tt, ptype, gtype, count):
    shapes = [SIZES[i % len(SIZES)] for i in range(count)]
    params = [rand(s, ptype, i).cuda() for i, s in enumerate(shapes)]
    opt = tt.AdamW(params, **HYPER)
    for t in (1, 2, 3):
        grads = [rand(s, gtype, 100 * t + i, 0.1).cuda() for i, s in enumerate(shapes)]
        before = [p.clone() for p in params]
        m0, v0 = ([x.clone() for x in s] for s in opt.state_values())
        opt.step(grads)
        m1, v1 = opt.state_values()
        for p, g, q, a, b, x, y in zip(before, grads, params, m0, v0, m1, v1):
            want, tol = formula64(p, g, a, b, t, HYPER, ptype)
            for got, w, e in zip((q, x, y), want, tol):
                assert got.shape == w.shape and ((got.double() - w).abs() <= e).all()
    assert opt.steps == 3


def philox_words(words, step, seed, salt=0x41444D57):
    """Philox4x32-10 on counters (i, i >> 32, step, salt): uint64 arrays [words, 4]."""
    low = np.uint64(0xFFFFFFFF)
    i = np.arange(words, dtype=np.uint64)
    c = [i & low, i >> np.uint64(32), np.full_like(i, step), np.full_like(i, salt)]
    k0, k1 = seed & 0xFFFFFFFF, seed >> 32
    for _ in range(10):
        a, b = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        c = [(b >> np.uint64(32)) ^ c[1] ^ np.uint64(k0), b & low, (a >> np.uint64(32)) ^ c[3] ^ np.uint64(k1), a & low]
        k0, k1 = (k0 + 0x9E3779B9) & 0xFFFFFFFF, (k1 + 0xBB67AE85) & 0xFFFFFFFF
    return np.stack(c, 1)


def plain_codes(m, v, step, seed):
    """Codes and scales of flat float32 moments (numpy float32 operations are IEEE), the rule of the C header."""
    f = np.float32
    w = philox_words(m.size // 4, step, seed).reshape(-1, 256)
    um = ((w & np.uint64(0xFFFF)).astype(f) + f(0.5)) * f(2.0**-16)
    uv = ((w >> np.uint64(16)).astype(f) + f(0.5)) * f(2.0**-16)
    m, v = m.reshape(-1, 256), v.reshape(-1, 256)
    tv = v.max(1)
    tv[tv < f(2.0**-90)] = 0
    tm = np.abs(m).max(1)
    tm[(tm < f(2.0**-100)) | (tv == 0)] = 0

    def encode(x, top, power, largest, u):
        inv = np.zeros_like(top)
        inv[top > 0] = f(float(largest**power)) / top[top > 0]
        y = x * inv[:, None]
        grid = (np.arange(largest + 2, dtype=np.float64) ** power).astype(f)
        k = np.searchsorted(grid[: largest + 1], y.ravel(), side="right").reshape(y.shape) - 1
        up = u * (grid[k + 1] - grid[k]) < y - grid[k]
        return y, k, np.minimum(k + up, largest)

    _, _, qm = encode(np.abs(m), tm, 2, 127, um)
    y, k, qv = encode(v, tv, 4, 255, uv)
    qv = np.where(k == 0, (y > 0).astype(qv.dtype), qv)
    return np.where(m < 0, -qm, qm).ravel(), qv.ravel(), tm, tv


def plain_values(qm, qv, tm, tv):
    f = np.float32
    c, d = qm.astype(f).reshape(-1, 256), qv.astype(f).reshape(-1, 256)
    d2 = d * d
    return ((c * np.abs(c)) * (tm * f(1 / 127**2))[:, None]).ravel(), ((d2 * d2) * (tv * f(1 / 255**4))[:, None]).ravel()


@pytest.mark.parametrize("ptype,gtype", TYPES)
@pytest.mark.parametrize("seed", [0, 0x9876543210FEDCBA])
def test_coded_moments_bit_for_bit(tt, ptype, gtype, seed):
    shapes = SIZES + [(1000, 33)]
    params = [rand(s, ptype, i, 0.1).cuda() for i, s in enumerate(shapes)]
    opt = tt.AdamW(params, state_bits=8, seed=seed, **HYPER)
    f, (b1, b2) = np.float32, HYPER["betas"]
    for t in (1, 2, 3, 4):
        # gradients of very different sizes within a block, zeros among them
        grads = [(rand(s, F32, 100 * t + i) * 10.0 ** rand(s, F32, 7 * i).clamp(-3, 1)).to(gtype) for i, s in enumerate(shapes)]
        grads = [torch.where(rand(s, F32, i + 50) > 1.5, torch.zeros(()), g.float()).to(gtype) for i, (s, g) in enumerate(zip(shapes, grads))]
        st = opt.state_dict()
        before = [p.clone().cpu() for p in params]
        opt.step([g.cuda() for g in grads])
        now = opt.state_dict()
        m, v = plain_values(*(st[k].cpu().numpy() for k in ("exp_avg", "exp_avg_sq", "exp_avg_scale", "exp_avg_sq_scale")))
        flat = np.zeros(opt.elements, f)
        for g, o in zip(grads, opt.offsets):
            flat[o : o + g.numel()] = g.float().numpy().ravel()
        m1 = m * f(b1) + flat * f(1 - b1)
        v1 = v * f(b2) + (flat * flat) * f(1 - b2)
        qm, qv, tm, tv = plain_codes(m1, v1, t, seed)
        assert now["step"] == t
        for name, want in (("exp_avg", qm), ("exp_avg_sq", qv), ("exp_avg_scale", tm), ("exp_avg_sq_scale", tv)):
            assert np.array_equal(now[name].cpu().numpy(), want), name
        vm, vv = opt.state_values(flat=True)
        wm, wv = plain_values(qm, qv, tm, tv)
        assert np.array_equal(vm.cpu().numpy(), wm) and np.array_equal(vv.cpu().numpy(), wv)
        # the step itself uses the moments before they are coded
        for p, q, g, o in zip(before, params, grads, opt.offsets):
            a, b = (torch.from_numpy(x[o : o + p.numel()].reshape(p.shape).copy()) for x in (m, v))
            want, tol = formula64(p, g, a, b, t, HYPER, ptype, 13.1)
            assert ((q.cpu().double() - want[0]).abs() <= tol[0]).all()


def test_many_coded_moments_bit_for_bit(tt):
    """Rare ties between a random word and a remainder: three million codes of each kind, twice."""
    n, f, (b1, b2) = 3_000_000, np.float32, HYPER["betas"]
    p = torch.zeros(n, device="cuda")
    opt = tt.AdamW([p], state_bits=8, seed=77, **HYPER)
    names = ("exp_avg", "exp_avg_sq", "exp_avg_scale", "exp_avg_sq_scale")
    for t in (1, 2):
        g = rand((n,), F32, t)
        st = opt.state_dict()
        opt.step([g.cuda()])
        now = opt.state_dict()
        m, v = plain_values(*(st[k].cpu().numpy() for k in names))
        flat = np.zeros(opt.elements, f)
        flat[:n] = g.numpy()
        want = plain_codes(m * f(b1) + flat * f(1 - b1), v * f(b2) + (flat * flat) * f(1 - b2), t, 77)
        for name, w in zip(names, want):
            assert np.array_equal(now[name].cpu().numpy(), w), name


def test_coded_moments_keep_their_mean(tt):
    """Averages whose step is far below a code's step still follow: constant gradients of several sizes in one block,
    v and m against their closed forms.  The mean over n equal elements of a value rounded at random, t times,
    scatters with at most sqrt(0.5 / (1 - b)) single steps of at most s = 4 / q (v) or 2 / q (m) relative, q the code
    of the value; six standard deviations over n elements, and the chain of float32 roundings far below."""
    n, t = 60 * 256, 200
    # each block: 200 elements of 0.3, 55 of 1 and one of 1.2; q of 0.3^2 / 1.2^2: 255 * 0.5 = 127; m: 127 * 0.5 = 63
    g = torch.full((n // 256, 256), 0.3)
    g[:, 200:] = 1.0
    g[:, 255] = 1.2
    p = torch.zeros(n, device="cuda")
    opt = tt.AdamW([p], state_bits=8, lr=0.0, betas=(0.9, 0.999), seed=5)
    grads = [g.reshape(-1).cuda()]
    for _ in range(t):
        opt.step(grads)
    m, v = (x.reshape(-1, 256)[:, :200].double().mean().item() for x in opt.state_values(flat=True))
    wm, wv = 0.3 * (1 - 0.9**t), 0.09 * (1 - 0.999**t)
    k = n // 256 * 200
    assert abs(v / wv - 1) < 6 * (4 / 127) * math.sqrt(0.5 * min(t, 1 / (1 - 0.999))) / math.sqrt(k)
    assert abs(m / wm - 1) < 6 * (2 / 63) * math.sqrt(0.5 / (1 - 0.9)) / math.sqrt(k)


@pytest.mark.parametrize("bits", [8, 32])
def test_views_orders_and_alignment(tt, bits):
    """Parameters and gradients at odd addresses and in other dimension orders step as their plain copies do."""
    def build():
        a = rand((4000,), BF16, 1).cuda()
        b = rand((37, 53), F32, 2).cuda()
        c = rand((6, 5, 9), F16, 3).cuda()
        return a, b, c

    a, b, c = build()
    odd = [a[3:1500], a[1501:3999], b.t(), c.permute(2, 0, 1)]
    a2, b2, c2 = build()
    plain = [a2[3:1500].clone(), a2[1501:3999].clone(), b2.t().clone(memory_format=torch.preserve_format), c2.permute(2, 0, 1).clone(memory_format=torch.preserve_format)]
    g = [rand((2001,), F32, 5).cuda()[1:1498], rand((2500,), BF16, 6).cuda()[2:], rand((37, 53), F32, 7).cuda().t(), rand((6, 5, 9), F16, 8).cuda().permute(2, 0, 1)]
    h = dict(lr=1e-2, state_bits=bits, seed=1)
    o1, o2 = tt.AdamW(odd, **h), tt.AdamW(plain, **h)
    for _ in range(3):
        o1.step(g)
        o2.step([x.clone(memory_format=torch.preserve_format) for x in g])
    for x, y in zip(odd, plain):
        assert torch.equal(x, y)
    for s1, s2 in zip(o1.state_values(), o2.state_values()):
        for x, y, p in zip(s1, s2, odd):
            assert torch.equal(x, y) and x.shape == p.shape and x.stride() == p.stride()
    # between and beside the views: untouched
    assert torch.equal(a[:3], a2[:3]) and torch.equal(a[1500:1501], a2[1500:1501]) and torch.equal(a[3999:], a2[3999:])


@pytest.mark.parametrize("bits", [8, 32])
def test_more_tensors_than_one_launch_holds(tt, bits):
    n = 1501
    params = [rand((1 + i % 7,), F32, i).cuda() for i in range(n)]
    ref = torch.cat([p for p in params])
    grads = [rand((1 + i % 7,), F32, 5000 + i).cuda() for i in range(n)]
    opt = tt.AdamW(params, state_bits=bits, **HYPER)
    for t in (1, 2):
        m, v = (torch.cat(x) for x in opt.state_values())
        opt.step(grads)
        (want, *_), (tol, *_) = formula64(ref, torch.cat(grads), m, v, t, HYPER, F32, 13.1)
        got = torch.cat(params)
        assert ((got.double() - want).abs() <= tol).all()
        ref = got
    assert opt.steps == 2


@pytest.mark.parametrize("bits", [8, 32])
def test_replayed_graph_counts_on_and_follows_lr(tt, bits):
    def run(capture):
        params = [rand((300, 7), BF16, 1).cuda(), rand((5,), F32, 2).cuda()]
        grads = [rand((300, 7), BF16, 3).cuda(), rand((5,), F32, 4).cuda()]
        opt = tt.AdamW(params, state_bits=bits, seed=3, **HYPER)
        opt.step(grads)
        if capture:
            graph = torch.cuda.CUDAGraph()
            with nat.capturing(graph):
                opt.step(grads)
        for k in range(6):
            if k == 3:
                opt.lr = 1e-4
            grads[0].mul_(0.5)
            graph.replay() if capture else opt.step(grads)
        torch.cuda.synchronize()
        return params, opt.state_dict()

    (p1, s1), (p2, s2) = run(False), run(True)
    assert all(torch.equal(a, b) for a, b in zip(p1, p2))
    assert s1["step"] == s2["step"] == 7 and all(torch.equal(s1[k], s2[k]) for k in s1 if k != "step")


@pytest.mark.parametrize("bits", [8, 32])
def test_state_dict_resumes_bit_for_bit(tt, bits):
    def fresh():
        return [rand((777,), F32, 1).cuda(), rand((30, 30), BF16, 2).cuda()]

    grads = [[rand((777,), F32, 10 + t).cuda(), rand((30, 30), BF16, 20 + t).cuda()] for t in range(4)]
    a = fresh()
    oa = tt.AdamW(a, state_bits=bits, seed=9, **HYPER)
    for g in grads[:2]:
        oa.step(g)
    b = [x.clone() for x in a]
    ob = tt.AdamW(b, state_bits=bits, seed=9, **HYPER)
    ob.load_state_dict(oa.state_dict())
    for g in grads[2:]:
        oa.step(g)
        ob.step(g)
    assert all(torch.equal(x, y) for x, y in zip(a, b)) and ob.steps == 4


def test_values_that_are_not_finite(tt):
    """float32 moments: element by element, as the formula has it.  Codes share a block's scale: the moments of the
    block become NaN, the parameters beside the bad element are stepped as usual in that step."""
    for bits in (32, 8):
        p = torch.ones(1024, device="cuda")
        g = torch.full((1024,), 0.5, device="cuda")
        g[300], g[301] = float("nan"), float("inf")
        g[900:] = 0.0
        opt = tt.AdamW([p], state_bits=bits, **HYPER)
        opt.step([g])
        bad = torch.zeros(1024, dtype=torch.bool, device="cuda")
        bad[300:302] = True
        assert torch.equal(~torch.isfinite(p), bad)
        m, v = opt.state_values(flat=True)
        if bits == 32:
            assert torch.equal(~torch.isfinite(m), bad) and torch.equal(~torch.isfinite(v), bad)
        else:
            block = torch.arange(1024, device="cuda") // 256 == 1
            assert torch.equal(torch.isnan(m), block) and torch.equal(torch.isnan(v), block)


def test_tiny_and_zero_gradients(tt):
    p = torch.ones(512, device="cuda")
    g = torch.zeros(512, device="cuda")
    g[256:] = 1e-18  # v = 1e-38: below what a block's scale holds
    opt = tt.AdamW([p], state_bits=8, lr=0.1, weight_decay=0.0)
    for _ in range(3):
        opt.step([g])
    assert torch.isfinite(p).all() and (p[:256] == 1).all()
    m, v = opt.state_values(flat=True)
    assert not m.any() and not v.any()
    # 20 orders of magnitude within a block: no element's v falls to zero
    g = torch.logspace(-10, 10, 512, device="cuda")
    p = torch.zeros(512, device="cuda")
    opt = tt.AdamW([p], state_bits=8, lr=0.1)
    for _ in range(20):
        opt.step([g])
    assert (opt.state_values(flat=True)[1] > 0).all() and torch.isfinite(p).all() and p.abs().max() < 20 * 0.1 * 8


def test_autograd_sees_the_update_and_grad_is_the_default(tt):
    w = torch.nn.Parameter(rand((40, 30), F32, 1).cuda())
    x = rand((8, 30), F32, 2).cuda().requires_grad_(True)  # so that the product saves w
    opt = tt.AdamW([w], lr=0.05, weight_decay=0.0)
    y = (x @ w.t()).square()
    version = w._version
    y.sum().backward()
    opt.step()
    assert w._version > version
    z = (x @ w.t()).square().sum()
    opt.step()
    with pytest.raises(RuntimeError):  # w changed after it was saved for the backward pass
        z.backward()


def test_refusals(tt):
    p = torch.zeros(10, device="cuda")
    for params, kw, exc in [
        ([], {}, ValueError),
        ([torch.zeros(3)], {}, ValueError),
        ([p.double()], {}, ValueError),
        ([p[::2]], {}, ValueError),
        ([p[:1].expand(4)], {}, ValueError),
        ([p, p[5:]], {}, ValueError),
        ([p], {"state_bits": 16}, ValueError),
        ([p], {"betas": (0.9, 1.0)}, ValueError),
        ([p], {"eps": 0.0}, ValueError),
        ([p], {"lr": -1.0}, ValueError),
        ([3], {}, (TypeError, ValueError)),
    ]:
        with pytest.raises(exc):
            tt.AdamW(params, **kw)
    q = torch.zeros((4, 6), device="cuda", dtype=torch.bfloat16)
    opt = tt.AdamW([p, q])
    good = [torch.ones_like(p), torch.ones_like(q)]
    for grads, exc in [
        (good[:1], ValueError),
        ([good[0], None], ValueError),
        ([good[0], good[1].half()], ValueError),
        ([good[0], good[1].cpu()], ValueError),
        ([good[0][:9], good[1]], ValueError),
        ([good[0], torch.ones((6, 4), device="cuda", dtype=torch.bfloat16).t()], ValueError),
        (None, ValueError),
    ]:
        with pytest.raises(exc):
            opt.step(grads)
    assert opt.steps == 0 and not p.any()
    opt.step(good)
    with pytest.raises(ValueError):
        opt.load_state_dict({"step": 1, "exp_avg": opt.exp_avg})
    with pytest.raises(ValueError):
        opt.load_state_dict({**opt.state_dict(), "exp_avg": torch.zeros(3, device="cuda")})
    with pytest.raises(ValueError):
        opt.lr = -1
