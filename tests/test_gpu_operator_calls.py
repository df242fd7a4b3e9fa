"""Calls of the operators around dense programs that their documentation allows beside the ordinary ones."""

import subprocess
import sys
from pathlib import Path

import numpy as np
import pytest
import torch
import torch.autograd.forward_ad as fw

from test_gpu_adamw import formula64
from tt_thrml_b200 import Executor, _native as nat, make_cuda_config, workloads
from tt_thrml_b200.core import Family

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


FRESH = """
import sys
sys.path[:0] = {paths!r}
import torch, tt_thrml_b200 as tt
from test_gpu_int8 import check_product, plain_quantize, rand
for kind in (torch.float32, torch.bfloat16, torch.float16, torch.int8):
    for rows, cols in {sizes!r}:
        w = rand((5, cols), torch.float32, cols)
        wq, sw = plain_quantize(w)
        x = rand((rows, cols), torch.float32 if kind == torch.int8 else kind, rows)
        weights = tt.QuantizedRows(torch.from_numpy(wq).to(torch.int8).cuda(), torch.from_numpy(sw).cuda())
        y = tt.int8_product(tt.quantize_rows(x.cuda()) if kind == torch.int8 else x.cuda(), weights)
        check_product(y, *plain_quantize(x), wq, sw, None, y.dtype)
"""


@pytest.mark.parametrize("sizes", [((1, 49152), (2, 24576)), ((1, 49089), (2, 24545)), ((1, 49120), (2, 24560))])
def test_rows_that_fill_48_kilobytes_of_shared_memory(sizes):
    """One and two rows around the shared memory that a launch has without asking for more, in a process that has not
    launched longer rows before (they raise the limit for later calls)."""
    root = Path(__file__).resolve().parents[1]
    code = FRESH.format(paths=[str(root), str(root / "tests")], sizes=sizes)
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stdout + r.stderr


def rbm():
    return workloads.gaussian_bernoulli_rbm(256, 512, seed=2, w_std=0.05)


@pytest.mark.parametrize("pinned", [True, False])
def test_a_host_batch_may_be_filled_anew_at_once(tt, pinned):
    """The learner's stream is busy while step() is called; the batch is overwritten as soon as it returns."""
    learner = tt.DenseLearner(rbm(), n_data=128, n_chains=128, config=make_cuda_config(dense_precision="fp32"))
    g = torch.Generator().manual_seed(1)
    staging = torch.empty((128, 256), pin_memory=pinned)
    for _ in range(3):
        rows = torch.randn((128, 256), generator=g)
        staging.copy_(rows)
        with torch.cuda.stream(learner.data.stream):
            torch.cuda._sleep(100_000_000)  # about 50 ms
        learner.step(staging)
        staging.fill_(7.0)
        assert np.array_equal(learner.data.raw_state()[:256].T, rows.numpy())


def loaded(program, config, chains=128, device=None):
    ex = Executor(None, device, program, config, n_chains=chains)
    g = torch.Generator().manual_seed(3)
    ex.load_state([torch.randn((chains, 256), generator=g), torch.randint(0, 2, (chains, 512), generator=g).bool()], [])
    return ex


def outputs_of(tt, operator):
    """A call that writes the tensors it is given, and their shapes."""
    if operator == "int8":
        w, x = tt.quantize_rows(torch.ones((4, 64), device="cuda")), torch.ones((2, 64), device="cuda")
        return (lambda o: tt.int8_product(x, w, out=o[0])), [(2, 4)]
    if operator == "moments":
        x, y = torch.ones((4, 5), dtype=BF16, device="cuda"), torch.ones((4, 6), dtype=BF16, device="cuda")
        return (lambda o: tt.pair_moments(x, y, out=tuple(o), units=True)), [(5, 6), (5,), (6,)]
    ex = loaded(rbm(), make_cuda_config(dense_precision="int8"))
    return (lambda o: ex.dense_moments(out=tuple(o), accumulate=True)), [(256, 512), (256,), (512,)]


@pytest.mark.parametrize("operator", ["int8", "moments", "dense"])
def test_autograd_sees_that_an_output_was_written(tt, operator):
    call, shapes = outputs_of(tt, operator)
    for i in range(len(shapes)):
        outs = [torch.zeros(s, device="cuda") for s in shapes]
        leaf = torch.ones(shapes[i], device="cuda", requires_grad=True)
        saved = (leaf * outs[i]).sum()
        call(outs)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            saved.backward()


@pytest.mark.parametrize("operator", ["int8", "moments", "dense"])
def test_outputs_that_require_a_gradient_are_refused(tt, operator):
    call, shapes = outputs_of(tt, operator)
    for i in range(len(shapes)):
        outs = [torch.zeros(s, device="cuda") for s in shapes]
        outs[i].requires_grad_(True)
        with pytest.raises(RuntimeError, match="requires a gradient"):
            call(outs)
        assert not any(o.detach().any() for o in outs)
        with torch.no_grad():
            call(outs)


def test_outputs_that_share_memory_are_refused(tt):
    x = torch.ones((4, 6), dtype=BF16, device="cuda")
    out, s = torch.zeros((6, 6), device="cuda"), torch.zeros(6, device="cuda")
    for outs in ((out, s, s), (out, out[1], s), (out, s, out[5])):
        with pytest.raises(ValueError, match="share memory"):
            tt.pair_moments(x, x, out=outs, units=True)
    ex = loaded(rbm(), make_cuda_config())
    out, s = torch.zeros((256, 512), device="cuda"), torch.zeros(512, device="cuda")
    for outs in ((out, s[:256], s), (out, out[0, :256], s)):
        with pytest.raises(ValueError, match="share memory"):
            ex.dense_moments(out=outs)
    torch.cuda.synchronize()
    assert not out.any() and not s.any()


@pytest.mark.parametrize("derivative", ["gradient", "tangent"])
def test_derivatives_are_not_dropped(tt, derivative):
    """Every input that a derivative could be asked of, from the first call and in the plain case after it."""
    r, m = tt.quantize_rows(torch.ones((4, 64), device="cuda")), torch.ones((4, 5), dtype=BF16, device="cuda")
    x, bias = torch.ones((2, 64), device="cuda"), torch.ones(4, device="cuda")
    tt.int8_product(x, r)
    tt.pair_moments(m, m)
    out = torch.zeros((2, 4), device="cuda")
    with fw.dual_level():
        def d(t):
            return t.clone().requires_grad_(True) if derivative == "gradient" else fw.make_dual(t.clone(), torch.ones_like(t))

        calls = {
            "x": lambda: tt.int8_product(d(x), r),
            "x, strided": lambda: tt.int8_product(d(x.repeat(1, 2))[:, ::2], r),
            "x, given output": lambda: tt.int8_product(d(x), r, out=out),
            "bias": lambda: tt.int8_product(x, r, bias=d(bias)),
            "scale": lambda: tt.int8_product(x, tt.QuantizedRows(r.values, d(r.scale))),
            "scale, given output": lambda: tt.int8_product(x, tt.QuantizedRows(r.values, d(r.scale)), out=out),
            "scale of x": lambda: tt.int8_product(tt.QuantizedRows(r.values, d(r.scale)), r),
            "rows": lambda: tt.quantize_rows(d(x)),
            "moments of x": lambda: tt.pair_moments(d(m), m),
            "moments of y": lambda: tt.pair_moments(m, d(m), units=True),
            "moments, given output": lambda: tt.pair_moments([m, d(m)], [m, m], out=torch.zeros((5, 5), device="cuda")),
        }
        for name, call in calls.items():
            with pytest.raises(RuntimeError, match="requires a gradient" if derivative == "gradient" else "tangent"):
                call()
                pytest.fail(name)
        if derivative == "gradient":
            with torch.no_grad():
                for call in calls.values():
                    call()
    assert tt.int8_product(x, r).requires_grad is False


@pytest.mark.parametrize("precision", ["bf16", "fp32", "int8"])
@pytest.mark.parametrize("device", ["cuda", "cpu"])
def test_a_batch_that_requires_a_gradient_leaves_no_graph(tt, precision, device):
    def run(requires_grad):
        learner = tt.DenseLearner(rbm(), n_data=128, n_chains=128, config=make_cuda_config(dense_precision=precision))
        g = torch.Generator().manual_seed(5)
        for _ in range(2):
            batch = torch.randn((128, 256), generator=g).to(device).requires_grad_(requires_grad)
            gradient = learner.step(batch * 1.0)
            assert not any(t.requires_grad for t in (*gradient, *learner.data._block_states))
        return learner.data.raw_state(), learner.weights.cpu()

    (s1, w1), (s2, w2) = run(False), run(True)
    assert np.array_equal(s1, s2) and torch.equal(w1, w2)


@pytest.mark.parametrize("bits", [8, 32])
@pytest.mark.parametrize("beta2", [0.999, 0.5, 0.9999999])
@pytest.mark.parametrize("eps", [1e-30, 1e-20, 1e-18, 1e-12, 4e-10, 5e-10, 1e-8])
def test_tiny_gradients_with_tiny_eps(tt, bits, eps, beta2):
    """Second moments below the smallest normal float32, some below the smallest subnormal: the update is the formula's
    for every eps that is allowed.  The computed v lies within ev of v1 (formula64: its roundings and 1e-44 for
    subnormal ones), not below 0, and the root, the denominator and the quotient are monotonic in it, so the
    update lies between those of v1 - ev and v1 + ev, less and more the 13.1 roundings of the coded steps elsewhere.
    (Where v1 <= ev, float32 need not hold v at all and m / eps is within this bound; elsewhere it is narrow.)"""
    g = torch.Generator().manual_seed(1)
    grads = torch.randn(4000, generator=g) * 10.0 ** (torch.rand(4000, generator=g) * 6 - 23)
    h = dict(lr=1e-3, betas=(0.9, beta2), eps=eps, weight_decay=0.0)
    p, zero = torch.zeros(4000, device="cuda"), torch.zeros(4000)
    opt = tt.AdamW([p], state_bits=bits, **h)
    opt.step([grads.cuda()])
    (_, m1, v1), (_, em, ev) = formula64(zero, grads, zero, zero, 1, h, F32)
    step, r = 1e-3 / (1 - 0.9), (1 - beta2) ** -0.5
    least = step * (m1.abs() - em) / ((v1 + ev).sqrt() * r + eps) * (1 - 14.1 * 2.0**-24)
    most = step * (m1.abs() + em) / ((v1 - ev).clamp_min(0).sqrt() * r + eps) * (1 + 14.1 * 2.0**-24)
    got = -p.cpu().double() * grads.sign()
    assert ((least <= got) & (got <= most)).all()
    narrow = v1 > 4 * ev  # the bound says something there
    assert narrow.sum() > 500 and (most[narrow] < 1.4 * least[narrow]).all()


def test_a_learner_reports_expired_waits(tt):
    """The words are set from the host, as a kernel that gives up sets them."""
    from tt_thrml_b200 import quantized

    learner = tt.DenseLearner(rbm(), n_data=128, n_chains=128)
    learner.step(torch.zeros((128, 256)))
    learner.check()
    for word in (quantized.error_word(learner.weights.device), learner.model._error_word, learner.data._error_word):
        word.fill_(2)
        with pytest.raises(RuntimeError, match="expired wait"):
            learner.check()
        word.zero_()
        torch.cuda.synchronize()
        learner.check()
    quantized.error_word(learner.weights.device).fill_(2)
    with pytest.raises(RuntimeError, match="expired wait"):
        tt.check_operator_errors()
    tt.check_operator_errors()


@pytest.mark.parametrize("rows", [1, 2, 70])
def test_outputs_beside_their_inputs_in_one_matrix(tt, rows):
    """Ranges of columns that do not meet, as a program that concatenates keeps them."""
    g = torch.Generator().manual_seed(2)
    w = tt.quantize_rows(torch.randn((40, 64), generator=g).cuda())
    both = torch.zeros((rows, 112), device="cuda")
    x = torch.randn((rows, 64), generator=g).cuda()
    both[:, 40:104] = x
    assert tt.int8_product(both[:, 40:104], w, out=both[:, :40]).data_ptr() == both.data_ptr()
    assert torch.equal(both[:, :40], tt.int8_product(x, w)) and torch.equal(both[:, 40:104], x) and not both[:, 104:].any()
    with pytest.raises(ValueError, match="shares memory"):
        tt.int8_product(both[:, 39:103], w, out=both[:, :40])
    a, b = (torch.randint(-4, 5, (rows, n), generator=g).to(BF16).cuda() for n in (6, 10))
    buffer = torch.zeros((7, 16), device="cuda")
    outs = (buffer[:6, :10], buffer[6, 10:], buffer[6, :10])
    tt.pair_moments(a, b, out=outs, units=True)
    assert torch.equal(outs[0], a.float().t() @ b.float()) and not buffer[:6, 10:].any()
    assert torch.equal(outs[1], a.float().sum(0)) and torch.equal(outs[2], b.float().sum(0))


@pytest.mark.parametrize("precision", ["bf16", "fp32", "int8"])
def test_weights_of_any_strides(tt, precision):
    """Expanded, transposed and cut-out couplings become the operands that their contiguous copies become."""
    line = torch.linspace(-1, 1, 512, device="cuda")
    whole = torch.randn((600, 700), generator=torch.Generator().manual_seed(1)).cuda()
    a, b = (Executor(None, None, rbm(), make_cuda_config(n_chains=128, dense_precision=precision)) for _ in range(2))
    for w in (line.expand(256, 512), line[:256, None].expand(256, 512), line[:1].expand(256, 512), whole[:512, :256].t(),
              whole[3:259, 5:517], whole[::2, :][:256, 100:612]):
        a.update_dense_weights(w)
        b.update_dense_weights(w.clone(memory_format=torch.contiguous_format))
        for p, q in zip(a._plans(), b._plans()):
            assert torch.equal(p.weights_nk, q.weights_nk)
            assert p.w_scale is None or torch.equal(p.w_scale, q.w_scale)


def test_a_learning_rate_set_in_a_capture(tt):
    """It acts when the graph is replayed, and what is set outside acts at once, also where it is the same number."""
    p, g = torch.zeros(4, device="cuda"), [torch.ones(4, device="cuda")]
    opt = tt.AdamW([p], lr=0.5, betas=(0.0, 0.0), eps=1e-30, weight_decay=0.0)  # a step is -lr exactly

    def stepped(run):
        p.zero_()
        run()
        return -p[0].item()

    assert stepped(lambda: opt.step(g)) == 0.5
    graph = torch.cuda.CUDAGraph()
    with nat.capturing(graph):
        opt.lr = 0.25
        opt.step(g)
    assert stepped(lambda: opt.step(g)) == 0.5  # nothing was replayed yet
    opt.lr = 0.25
    assert stepped(lambda: opt.step(g)) == 0.25
    opt.lr = 0.125
    assert stepped(lambda: opt.step(g)) == 0.125
    assert stepped(graph.replay) == 0.25 and stepped(lambda: opt.step(g)) == 0.25
    opt.lr = 0.125
    assert stepped(lambda: opt.step(g)) == 0.125


def test_settings_that_are_fixed_cannot_be_set(tt):
    opt = tt.AdamW([torch.ones(4, device="cuda")], betas=(0.5, 0.75), eps=1e-6, weight_decay=0.25, state_bits=8, seed=3)
    for name, value in (("betas", (0.5, 0.75)), ("eps", 1e-6), ("weight_decay", 0.25), ("state_bits", 8), ("seed", 3)):
        assert getattr(opt, name) == value
        with pytest.raises(AttributeError):
            setattr(opt, name, value)
    opt.params.append(torch.ones(4, device="cuda"))
    with pytest.raises(ValueError, match="made for 1"):
        opt.step([torch.ones(4, device="cuda")] * 2)
    assert opt.steps == 0


@pytest.mark.parametrize("precision", ["bf16", "int8"])
def test_shared_weights_of_an_executor_that_shares_a_third_ones(tt, precision):
    """Sharing goes along chains, through captured sweeps too, and ends where an executor shares another one's."""
    cfg, dev = make_cuda_config(dense_precision=precision), tt.open_device(device_id=0)
    a, b, c, d = (loaded(rbm(), cfg, device=dev) for _ in range(4))
    weights = [torch.from_numpy(workloads.gaussian_bernoulli_rbm(256, 512, seed=k, w_std=0.05).W).cuda() for k in range(4)]

    def same(x, y):
        assert all(p.weights_nk is q.weights_nk and p.w_scale is q.w_scale and p.bias is q.bias for p, q in zip(x._plans(), y._plans()))
        states = []
        for ex in (x, y):
            ex.set_raw_state(start)
            ex.prepare_rng(4)
            ex.run_sweeps(3)
            states.append(ex.raw_state())
        assert np.array_equal(*states)

    start = a.raw_state()
    a.share_dense_weights(b)
    b.update_dense_weights(weights[0])
    same(a, b)  # their sweeps are captured now
    b.share_dense_weights(c)
    same(a, c)
    c.update_dense_weights(weights[1])
    same(a, c)
    same(b, c)
    b.update_dense_weights(weights[2])  # writes what all three run on
    same(a, c)
    a.share_dense_weights(d)
    d.update_dense_weights(weights[3])
    same(a, d)
    same(b, c)
    assert a._plans()[0].weights_nk is not b._plans()[0].weights_nk
    b.share_dense_weights(d)  # a no longer follows b, c never did
    same(a, b)
    assert c._plans()[0].weights_nk is not d._plans()[0].weights_nk
    d.share_dense_weights(a)  # a circle
    a.share_dense_weights(a)
    d.update_dense_weights(weights[0])
    same(a, d)


def test_host_batches_of_several_types_in_turn(tt):
    """Bools, floats and halves one after the other without waiting, each the data states of its step."""
    program = workloads.DenseBipartiteProgram(rbm().W, rbm().b_v, rbm().b_h, visible_family=Family.SPIN)
    g = torch.Generator().manual_seed(6)
    spins = [torch.randint(0, 2, (128, 256), generator=g).bool() for _ in range(9)]
    kinds = [torch.bool, F32, F32, torch.float16, torch.bool, F32, F32, F32, torch.float64]

    def run(to):
        learner = tt.DenseLearner(program, n_data=128, n_chains=128, config=make_cuda_config(dense_precision="int8"))
        gradients = []
        for s, kind in zip(spins, kinds):
            batch = s.clone() if kind == torch.bool else (s.to(kind) * 2 - 1)
            batch = to(batch)
            gradients.append([t.clone() for t in learner.step(batch)])
            if batch.device.type == "cpu":
                batch.zero_()
        return learner, gradients

    host, wanted = run(lambda t: t.pin_memory()), run(lambda t: t.cuda())
    for a, b in zip(host[1], wanted[1]):
        assert all(torch.equal(x, y) for x, y in zip(a, b))
    assert torch.equal(host[0].weights, wanted[0].weights)


@pytest.mark.parametrize("chains", [640, 2176])
def test_dense_moments_of_many_chains(tt, chains):
    """One MMA adds 16 products to its accumulator within 17 steps of 2^-23 of the sum of magnitudes; at most 64 of them (1024
    chains) follow each other before the sum moves to a float32 register, with a rounding for each further 1024 chains
    and for the parts of a split (8 at most); a value in three bf16 pieces adds its phases (6) and 2^-24 of itself."""
    ex = loaded(rbm(), make_cuda_config(dense_precision="fp32"), chains)
    state = ex.raw_state().astype(np.float64)
    v, h = state[:256], state[256:]
    got = ex.dense_moments(0.5)
    steps = 17 * min(64, -(-chains // 16)) + -(-chains // 1024) + 8 + 6 + 1
    for g, want, mags in zip(got, (v @ h.T, v.sum(1), h.sum(1)), (np.abs(v) @ np.abs(h).T, np.abs(v).sum(1), np.abs(h).sum(1))):
        # (the unit sums are float32 additions, half a step each: at most a sixteenth of the chains one after the other)
        assert (np.abs(g.double().cpu().numpy() - 0.5 * want) <= 0.5 * steps * 2.0**-23 * mags).all()


def test_second_moments_of_one_block_never_fall_to_zero(tt):
    """Gradients over 20 orders of magnitude, v over 40, within one block of 256 that shares a scale."""
    g = torch.logspace(-10, 10, 256, device="cuda")
    p = torch.zeros(256, device="cuda")
    opt = tt.AdamW([p], state_bits=8, lr=0.1)
    for _ in range(20):
        opt.step([g])
    m, v = opt.state_values(flat=True)
    assert (v > 0).all() and torch.isfinite(v).all() and torch.isfinite(m).all()
    assert torch.isfinite(p).all()
