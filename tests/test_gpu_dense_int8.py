"""Dense sweeps on 8-bit operands (dense_precision="int8"), replaced couplings, dense moments and the learner."""

import ctypes
import gc

import numpy as np
import pytest
import torch

from oracle import oracle as orc
from tt_thrml_b200 import BulkRNGBuffers, Executor, _native as nat, make_cuda_config, workloads
from tt_thrml_b200.core import Family

import gpu_harness as gh

pytestmark = pytest.mark.gpu
F = np.float32


def plain_quantize(x):
    top = np.abs(x).max(1)
    live = top >= F(2.0**-120)
    inv = np.zeros_like(top)
    inv[live] = F(127.0) / top[live]
    return np.clip(np.rint(x * inv[:, None]), -127, 127).astype(np.int64), np.where(live, top * F(1.0 / 127.0), F(0)).astype(F)


def plain_field(q, sx, w, sw, bias):
    """The float32 field [chains, units]: exact sum, then one rounding for its conversion, the scales' product, the
    scaling and the bias (numpy float32 operations are IEEE, as the kernel's are)."""
    acc = (q @ w.T).astype(F)
    f = acc * (sx[:, None] * sw[None, :])
    return f if bias is None else f + bias[None, :]


def call(q, sx, w, sw, bias, family, precision, *, row0=0, variates=None, seed=1, sweep=0, chain_offset=0, fill=0):
    C, K = q.shape
    N = w.shape[0]
    pitch = -(-K // 16) * 16

    def lay(x):
        t = torch.zeros((x.shape[0], pitch), dtype=torch.int8)
        t[:, :K] = torch.from_numpy(x.astype(np.int8))
        return t.cuda()

    out = torch.full((C + 3, N), fill, dtype=torch.int8 if family == nat.SPIN else torch.bfloat16, device="cuda")
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    held = [lay(q), lay(w), torch.from_numpy(sw).cuda()]
    opt = [None if t is None else torch.from_numpy(np.ascontiguousarray(t)).cuda() for t in (sx, bias, variates)]
    p = [None if t is None else t.data_ptr() for t in opt]
    nat.bind_device(0)
    lib = nat.lib()
    rc = lib.tthrml_int8_field_sample(
        held[0].data_ptr(), pitch, p[0], held[1].data_ptr(), pitch, held[2].data_ptr(), C, N, K, p[1], family,
        ctypes.c_float(precision), out.data_ptr(), row0, chain_offset, p[2], 0 if variates is None else variates.shape[0],
        seed, sweep, None, err.data_ptr(), torch.cuda.current_stream().cuda_stream,
    )
    assert rc == 0, lib.tthrml_last_error()
    torch.cuda.synchronize()
    assert int(err.item()) == 0
    assert (out[C:] == fill).all()  # the rows behind the last chain: as they were
    return out[:C].float().cpu().numpy()


def operands(C, N, K, seed, spins=False):
    r = np.random.default_rng(seed)
    q, sx = (r.integers(0, 2, (C, K)) * 2 - 1, None) if spins else plain_quantize(r.standard_normal((C, K)).astype(F))
    w, sw = plain_quantize((0.1 * r.standard_normal((N, K))).astype(F))
    return q, sx, w, sw, (0.3 * r.standard_normal(N)).astype(F), r


SHAPES = [(1, 32, 16), (128, 256, 64), (200, 288, 100), (256, 256, 256), (300, 64, 1000), (513, 800, 130)]


@pytest.mark.parametrize("spins", [True, False])
@pytest.mark.parametrize("C,N,K", SHAPES)
def test_spin_draws_with_variates_are_bit_exact(C, N, K, spins):
    q, sx, w, sw, bias, r = operands(C, N, K, C + N, spins)
    for b in (bias, None):
        logits = r.logistic(size=(2, N, C)).astype(F)
        got = call(q, sx, w, sw, b, nat.SPIN, 1.0, variates=logits, sweep=1, fill=5)
        f = plain_field(q, np.ones(C, F) if sx is None else sx, w, sw, b)
        want = np.where(F(2) * f - logits[1].T > 0, 1, -1)
        assert np.array_equal(got, want)


@pytest.mark.parametrize("precision", [1.0, 2.5])
@pytest.mark.parametrize("C,N,K", SHAPES)
def test_gaussian_draws_with_variates_are_bit_exact(C, N, K, precision):
    q, sx, w, sw, bias, r = operands(C, N, K, C + N + 1, spins=True)
    xi = r.standard_normal((1, N, C)).astype(F)
    got = call(q, sx, w, sw, bias, nat.GAUSSIAN, precision, variates=xi)
    inv = F(1) / (F(precision) + F(1e-6))
    v = plain_field(q, np.ones(C, F), w, sw, bias) * inv + np.sqrt(inv) * xi[0].T
    assert np.array_equal(got, torch.from_numpy(v).to(torch.bfloat16).float().numpy())


@pytest.mark.parametrize("C,N,K,row0,offset", [(300, 64, 256, 0, 0), (256, 288, 100, 512, 128), (130, 32, 48, 6, 4)])
def test_philox_draws_follow_the_threshold(C, N, K, row0, offset):
    q, sx, w, sw, bias, _ = operands(C, N, K, 3)
    seed, sweep = 0x1234567890ABCDEF, 9
    got = call(q, sx, w, sw, bias, nat.SPIN, 1.0, row0=row0, seed=seed, sweep=sweep, chain_offset=offset)
    f = plain_field(q, sx, w, sw, bias).astype(np.float64)
    rows = row0 + np.arange(N)
    t = np.empty((C, N))
    for c in range(C):
        for g in np.unique(rows // 4):
            words = orc.philox4x32_10([c + offset, int(g), sweep, 0x44535049], [seed & 0xFFFFFFFF, seed >> 32])
            for n in np.nonzero(rows // 4 == g)[0]:
                t[c, n] = (2 * (int(words[rows[n] % 4]) >> 9) + 1) * 2.0**-24
    t *= 1 + np.exp(-2 * f)
    # e^(-2 f) is off by |2 f| 2^-23 (its argument) + 2^-21 (the approximation), t by three more roundings: below 1e-5
    # of t while |f| < 20
    assert np.abs(f).max() < 20
    sure = np.abs(t - 1) > 1e-5
    assert sure.mean() > 0.999 and np.array_equal(got[sure], np.where(t < 1, 1, -1)[sure])


def test_gaussian_philox_draws_have_the_right_moments():
    C, N, K = 4096, 256, 32
    q, sx, w, sw, bias, _ = operands(C, N, K, 5, spins=True)
    got = call(q, sx, w, sw, bias, nat.GAUSSIAN, 4.0, seed=7)
    f = plain_field(q, np.ones(C, F), w, sw, bias)
    z = (got - f / 4.000001) * 2.0000002
    n = z.size
    # bf16 rounding adds at most (2^-8 |v|)^2 / 3 to the variance; |v| < 4
    assert abs(z.mean()) < 6 / np.sqrt(n) and abs(z.var() - 1) < 6 * np.sqrt(2 / n) + 4 * (2.0**-8 * 4) ** 2 / 3


def int8_executor(program, C, mode="philox", **kw):
    return Executor(None, None, program, make_cuda_config(n_chains=C, rng_mode=mode, dense_precision="int8", **kw), n_sweeps=8)


def rbm(spin_visible=False, seed=2):
    p = workloads.gaussian_bernoulli_rbm(256, 512, seed=seed, w_std=0.05)
    if not spin_visible:
        return p
    return workloads.DenseBipartiteProgram(p.W, p.b_v, p.b_h, visible_family=Family.SPIN)


@pytest.mark.parametrize("spin_visible", [False, True])
@pytest.mark.parametrize("C", [128, 384])
def test_executor_sweeps_group_by_group(C, spin_visible):
    program = rbm(spin_visible)
    ex = int8_executor(program, C, mode="parity")
    assert ex.compiled.state_dtype == "dense_int8"
    r = np.random.default_rng(4)
    v0 = r.integers(0, 2, (C, 256)).astype(bool) if spin_visible else r.standard_normal((C, 256)).astype(F)
    ex.load_state([v0, r.integers(0, 2, (C, 512)).astype(bool)], [])
    S = 3
    buffers, _ = gh.make_variates(ex, S)
    ex._install_rng(buffers, S)
    W = {0: plain_quantize(program.W), 1: plain_quantize(np.ascontiguousarray(program.W.T))}
    B = {0: program.b_v, 1: program.b_h}
    for sweep in range(S):
        for group in ex.compiled.sampling_groups:
            state = ex.raw_state()
            (bi,) = group.block_indices
            src = state[256:].T if bi == 0 else state[:256].T
            ex._run_sampling_group(group, sweep)
            now = ex.raw_state()
            gaussian_source = bi == 1 and not spin_visible
            q, sx = plain_quantize(np.ascontiguousarray(src)) if gaussian_source else (src.astype(np.int64), np.ones(C, F))
            f = plain_field(q, sx, *W[bi], B[bi])
            var = ex._variates(bi).cpu().numpy().reshape(S, -1, C)[sweep].T
            if bi == 0 and not spin_visible:
                inv = F(1) / (F(1) + F(1e-6))
                want = torch.from_numpy(f * inv + np.sqrt(inv) * var).to(torch.bfloat16).float().numpy()
            else:
                want = np.where(F(2) * f - var > 0, 1, -1)
            got = now[:256].T if bi == 0 else now[256:].T
            assert np.array_equal(got, want)
        ex._sweep_counter += 1
    ex.check_device_errors()
    assert ex.near_ties_dropped() == 0


@pytest.mark.parametrize("spin_visible", [False, True])
def test_graphs_checkpoints_and_readback(spin_visible, tmp_path):
    program, C = rbm(spin_visible), 256
    r = np.random.default_rng(1)
    init = [r.integers(0, 2, (C, 256)).astype(bool) if spin_visible else r.standard_normal((C, 256)).astype(F),
            r.integers(0, 2, (C, 512)).astype(bool)]

    def fresh(**kw):
        ex = int8_executor(program, C, **kw)
        ex.load_state(init, [])
        ex.prepare_rng(5)
        return ex

    a, b, c = fresh(), fresh(cuda_graphs=False), fresh()
    a.run_sweeps(6)
    b.run_sweeps(6)
    c.run_sweeps(2)
    c.save_checkpoint(tmp_path / "c.npz")
    d = int8_executor(program, C)
    d.load_checkpoint(tmp_path / "c.npz")
    d.run_sweeps(4)
    assert np.array_equal(a.raw_state(), b.raw_state()) and np.array_equal(a.raw_state(), d.raw_state())
    blocks = program.gibbs_spec.blocks
    seen = a.observe(blocks)
    assert seen[blocks[1]].dtype == np.bool_ and np.array_equal(seen[blocks[1]] * 2.0 - 1, a.raw_state()[256:].T)
    sums = a.block_sums([1])
    assert np.array_equal(sums, a.raw_state()[256:].astype(np.float64).sum(0))
    # another precision's checkpoint is another executor's
    e = Executor(None, None, program, make_cuda_config(n_chains=C), n_sweeps=8)
    with pytest.raises(ValueError):
        e.restore(c.checkpoint())


def test_a_capture_outlives_the_garbage_collector():
    """A CUDA graph in a reference cycle that becomes garbage before another capture is not freed within it."""
    ex = int8_executor(rbm(), 128)
    ex.load_state([np.zeros((128, 256), F), np.ones((128, 512), bool)], [])
    ex.prepare_rng(1)
    graph = torch.cuda.CUDAGraph()
    held = torch.zeros(8, device="cuda")
    with nat.capturing(graph):
        held.add_(1)
    cycle = [graph]
    cycle.append(cycle)
    del graph, cycle
    limits = gc.get_threshold()
    gc.set_threshold(1)  # collect at every chance
    try:
        ex.run_sweeps(4)
    finally:
        gc.set_threshold(*limits)
    ex.check_device_errors()
    assert gc.isenabled()


@pytest.mark.parametrize("precision", ["bf16", "fp32", "int8"])
@pytest.mark.parametrize("spin_visible", [False, True])
def test_replaced_weights_are_those_of_a_new_program(precision, spin_visible):
    C = 128
    old, new = rbm(spin_visible, 2), rbm(spin_visible, 3)
    new.b_h[:] = workloads.bf16_representable(np.linspace(-1, 1, 512).astype(F))
    cfg = make_cuda_config(n_chains=C, dense_precision=precision)
    init = [np.zeros((C, 256), F) + np.linspace(-1, 1, 256, dtype=F), np.ones((C, 512), bool)]

    def run(ex, n=3):
        ex.load_state(init, [])
        ex.prepare_rng(3)
        ex.run_sweeps(n)
        return ex.raw_state()

    first = Executor(None, None, old, cfg, n_sweeps=8)
    before = run(first)
    W, b0, b1 = (torch.from_numpy(np.ascontiguousarray(t)).cuda() for t in (new.W, new.b_v, new.b_h))
    first.update_dense_weights(W, b0, b1)
    W.zero_()  # the caller may change it at once
    after = run(first)
    assert np.array_equal(after, run(Executor(None, None, new, cfg, n_sweeps=8)))
    assert np.array_equal(before, run(Executor(None, None, old, cfg, n_sweeps=8)))  # the cached plan is as it was
    # in place from now on: the captured graph sees the next change
    first.update_dense_weights(torch.from_numpy(old.W).cuda(), torch.from_numpy(old.b_v).cuda(), torch.from_numpy(old.b_h).cuda())
    assert np.array_equal(run(first), before)


def test_refusals_of_weights_and_moments():
    ex = int8_executor(rbm(), 128)
    W = torch.zeros((256, 512), device="cuda")
    for args in [(W.half(),), (W.cpu(),), (W.t(),), (W, torch.zeros(3, device="cuda"))]:
        with pytest.raises(ValueError):
            ex.update_dense_weights(*args)
    with pytest.raises(RuntimeError):
        ex.dense_moments()  # no state
    sparse = Executor(None, None, workloads.erdos_renyi_ising(64, 4.0, seed=1), make_cuda_config(n_chains=32))
    with pytest.raises(NotImplementedError):
        sparse.update_dense_weights(W)
    with pytest.raises(NotImplementedError):
        sparse.dense_moments()
    with pytest.raises(ValueError):
        make_cuda_config(dense_precision="int4")


def moments64(state, scale):
    v, h = state[:256].astype(np.float64), state[256:].astype(np.float64)
    return scale * v @ h.T, scale * v.sum(1), scale * h.sum(1)


def close(got, want, state, scale, chains):
    """Within the float32 sums' bound: 17 steps of 2^-23 per MMA of 16 chains, at most 32 of them, of the sum of
    magnitudes, and one step per further addition; a value held in three pieces is exact but for float32."""
    mags = moments64(np.abs(state), abs(scale))
    steps = 17 * min(32, -(-chains // 16)) + chains // 512 + 24
    for g, w, m in zip(got, want, mags):
        assert (np.abs(g.double().cpu().numpy() - w) <= steps * 2.0**-23 * m + 1e-12).all()


@pytest.mark.parametrize("precision", ["bf16", "fp32", "int8"])
@pytest.mark.parametrize("spin_visible", [False, True])
def test_dense_moments_of_the_states(precision, spin_visible):
    C = 256
    ex = Executor(None, None, rbm(spin_visible), make_cuda_config(n_chains=C, dense_precision=precision), n_sweeps=8)
    r = np.random.default_rng(0)
    ex.load_state([r.standard_normal((C, 256)).astype(F), r.integers(0, 2, (C, 512)).astype(bool)], [])
    ex.prepare_rng(1)
    ex.run_sweeps(2)
    out = ex.dense_moments(0.5)
    state = ex.raw_state()
    close(out, moments64(state, 0.5), state, 0.5, C)
    again = ex.dense_moments(0.5, out=tuple(t.clone() for t in out), accumulate=True)
    for a, b in zip(again, out):
        assert torch.equal(a, b + b)


@pytest.mark.parametrize("precision", ["bf16", "fp32", "int8"])
@pytest.mark.parametrize("bits", [32, 8])
def test_learner_steps(precision, bits):
    """Two steps as they would be used: the gradient is the moment difference of the two executors' states, the masters
    take the AdamW step with it, and the samplers run on the new couplings."""
    import tt_thrml_b200 as tt

    program = rbm(seed=6)
    cfg = make_cuda_config(dense_precision=precision)
    h = dict(lr=1e-2, betas=(0.9, 0.99), weight_decay=0.01, state_bits=bits)
    learner = tt.DenseLearner(program, n_data=128, n_chains=256, config=cfg, sweeps=2, seed=4, **h)
    masters = [t.clone() for t in (learner.weights, learner.visible_bias, learner.hidden_bias)]
    shadow = tt.AdamW(masters, seed=4, eps=1e-8, **h)
    g = torch.Generator().manual_seed(1)
    for t in range(2):
        batch = torch.randn((128, 256), generator=g)
        gradient = learner.step(batch.cuda() if t else batch.pin_memory())
        torch.cuda.synchronize()
        sd, sm = learner.data.raw_state(), learner.model.raw_state()
        held = batch if precision == "fp32" else batch.to(torch.bfloat16).float()
        assert np.array_equal(sd[:256].T, held.numpy())
        want = [a + b for a, b in zip(moments64(sd, -1 / 128), moments64(sm, 1 / 256))]
        mags = [a + b for a, b in zip(moments64(np.abs(sd), 1 / 128), moments64(np.abs(sm), 1 / 256))]
        for got, w, m in zip(gradient, want, mags):
            assert (np.abs(got.double().cpu().numpy() - w) <= (17 * 16 + 60) * 2.0**-23 * m + 1e-12).all()
        shadow.step([x.clone() for x in gradient])
        for a, b in zip(masters, (learner.weights, learner.visible_bias, learner.hidden_bias)):
            assert torch.equal(a, b)
        for ex in (learner.data, learner.model):
            plans = sorted(ex._plans(), key=lambda p: p.block_indices[0])
            for plan, w, b in ((plans[0], learner.weights, learner.visible_bias), (plans[1], learner.weights.t(), learner.hidden_bias)):
                assert torch.equal(plan.bias, b)
                if precision == "int8":
                    q, s = plain_quantize(np.ascontiguousarray(w.cpu().numpy()))
                    assert np.array_equal(plan.weights_nk.cpu().numpy()[:, : w.shape[1]], q) and np.array_equal(plan.w_scale.cpu().numpy(), s)
                else:
                    for k in range(plan.source_pieces):
                        assert torch.equal(plan.weights_nk[:, k * w.shape[1] : (k + 1) * w.shape[1]], w.to(torch.bfloat16))
            ex.check_device_errors()
    tt.check_operator_errors()
    with pytest.raises(ValueError):
        learner.step(torch.zeros((64, 256)))


def test_mesh_of_one_and_shared_weights():
    """A MeshExecutor's 8-bit sweeps, weights and moments are its executor's; shared operands follow their owner."""
    import tt_thrml_b200 as tt

    program, C = rbm(), 128
    cfg = make_cuda_config(n_chains=C, dense_precision="int8")
    dev = tt.open_device(device_id=0)
    one, two = (Executor(None, dev, program, cfg, n_sweeps=8) for _ in range(2))
    mesh = tt.make_mesh_executor(None, dev, program, cfg, n_sweeps=8)
    W = torch.from_numpy(rbm(seed=9).W).cuda()
    one.update_dense_weights(W)
    two.share_dense_weights(one)
    mesh.update_dense_weights(W)
    one.update_dense_weights(W * 0.5)
    mesh.update_dense_weights(W * 0.5)
    init = [np.linspace(-1, 1, 256, dtype=F) + np.zeros((C, 1), F), np.ones((C, 512), bool)]
    states = []
    for ex in (one, two, mesh):
        ex.load_state(init, [])
        ex.prepare_rng(4)
        ex.run_sweeps(3)
        states.append(ex)
    assert np.array_equal(one.raw_state(), two.raw_state())
    assert np.array_equal(one.raw_state(), mesh.shards[0].raw_state())
    for a, b in zip(one.dense_moments(0.5), mesh.dense_moments(0.5)):
        assert torch.equal(a, b)
    with pytest.raises(NotImplementedError):
        mesh.share_dense_weights(one)
    apart = Executor(None, None, program, cfg, n_sweeps=8)
    with pytest.raises(ValueError):
        apart.share_dense_weights(one)
    with pytest.raises(ValueError):
        Executor(None, dev, program, make_cuda_config(n_chains=C, dense_precision="bf16")).share_dense_weights(one)


@pytest.mark.parametrize("precision", ["int8", "bf16"])
def test_weights_shared_before_the_first_update(precision):
    import tt_thrml_b200 as tt

    program, C = rbm(), 128
    cfg = make_cuda_config(n_chains=C, dense_precision=precision)
    dev = tt.open_device(device_id=0)
    one, two, other = (Executor(None, dev, program, cfg, n_sweeps=8) for _ in range(3))
    two.share_dense_weights(one)
    new = rbm(seed=9)
    one.update_dense_weights(torch.from_numpy(new.W).cuda(), torch.from_numpy(new.b_v).cuda())
    for p, q, kept in zip(one._plans(), two._plans(), other._plans()):
        assert p.weights_nk.data_ptr() == q.weights_nk.data_ptr() and p.bias.data_ptr() == q.bias.data_ptr()
        assert not torch.equal(p.weights_nk, kept.weights_nk)  # an executor that does not share keeps the program's
    init = [np.linspace(-1, 1, 256, dtype=F) + np.zeros((C, 1), F), np.ones((C, 512), bool)]
    for ex in (one, two):
        ex.load_state(init, [])
        ex.prepare_rng(4)
        ex.run_sweeps(3)
    assert np.array_equal(one.raw_state(), two.raw_state())


def test_learner_refusals():
    import tt_thrml_b200 as tt

    with pytest.raises(ValueError):
        tt.DenseLearner(rbm(), n_data=128, n_chains=128, sweeps=0)
    with pytest.raises(ValueError):
        tt.DenseLearner(rbm(), n_data=128, n_chains=128, config=make_cuda_config(rng_mode="parity"))
    with pytest.raises(NotImplementedError):  # 100 chains do not reach the dense kernels
        tt.DenseLearner(rbm(), n_data=100, n_chains=128)


def test_learner_on_spins_and_two_learners_at_once():
    """Spin batches (as bools or +-1), and two learners side by side: each its own streams, draws and operands."""
    import tt_thrml_b200 as tt

    g = torch.Generator().manual_seed(0)
    batch = torch.randint(0, 2, (128, 256), generator=g).bool()

    def make(seed):
        return tt.DenseLearner(rbm(True), n_data=128, n_chains=128, config=make_cuda_config(dense_precision="int8"), seed=seed)

    alone = [make(s) for s in (1, 2)]
    for ln in alone:
        for _ in range(3):
            ln.step(batch.cuda())
    both = [make(s) for s in (1, 2)]
    for _ in range(3):
        for ln in both:
            ln.step(batch.float().cuda() * 2 - 1)
    torch.cuda.synchronize()
    for a, b in zip(alone, both):
        assert torch.equal(a.weights, b.weights) and torch.equal(a.hidden_bias, b.hidden_bias)
    assert not torch.equal(both[0].weights, both[1].weights)
