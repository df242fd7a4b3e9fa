"""The categorical readout: dropout, cross entropy, AdamW and 4-bit fields as they are used together."""

import pytest
import torch

from test_gpu_dropout import plain as plain_dropout
from test_gpu_xent import close, expected
from tt_thrml_b200 import workloads

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def tt():
    import tt_thrml_b200

    return tt_thrml_b200


def data(rows, k, v, seed):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, k, generator=g).bfloat16().cuda()
    y = torch.randint(0, v, (rows,), generator=g)
    return x, torch.where(torch.rand(rows, generator=g) < 0.1, -100, y).cuda()


@pytest.mark.parametrize("rows,k,v,p", [(150, 72, 333, 0.0), (200, 64, 1000, 0.3), (5, 33, 17, 0.5)])
def test_a_step_has_the_gradient_of_the_formula(tt, rows, k, v, p):
    r = tt.CategoricalReadout(k, v, dropout=p, seed=3, lr=1e-2)
    for step in range(2):
        x, y = data(rows, k, v, step)
        units = plain_dropout(x.cpu(), p, 3, step).cuda() if p else x
        w, bias, before = r.weights.bfloat16(), r.bias.clone(), r.weights.clone()
        n = max(1, int((y != -100).sum()))
        weight = torch.full((rows,), 1.0 / n, device="cuda")
        (loss, dloss), _, (dw, dw_off), db = expected(units, w, y, bias, weight)
        got = r.step(x, y)
        total = loss.sum() / n
        close("loss", got, (total, dloss.sum() / n + 2.0**-22 * total.abs()))
        # float32 gradients: without the rounding to 16 bits that `expected` ends with
        close("dw", r.gradient[0], (dw, dw_off))
        close("db", r.gradient[1], db)
        assert not torch.equal(r.weights, before)
        assert torch.equal(r._operands, r.weights.bfloat16())
    r.check()


def test_a_captured_step_counts_on(tt):
    """Replayed steps are the eager ones, masks of the dropout included."""
    x, y = data(160, 48, 90, 7)

    def trained(captured):
        r = tt.CategoricalReadout(48, 90, dropout=0.4, seed=11, lr=1e-2)
        losses = [r.step(x, y).clone()]
        if not captured:
            losses += [r.step(x, y).clone() for _ in range(3)]
        else:
            side = torch.cuda.Stream()
            side.wait_stream(torch.cuda.current_stream())
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.stream(side), torch.cuda.graph(graph, stream=side):
                loss = r.step(x, y)
            for _ in range(3):
                graph.replay()
                torch.cuda.synchronize()
                losses.append(loss.clone())
        torch.cuda.synchronize()
        return losses, r.weights, r.bias

    a, b = trained(False), trained(True)
    for s, t in zip(a[0], b[0]):
        assert torch.equal(s, t)
    assert torch.equal(a[1], b[1]) and torch.equal(a[2], b[2])
    assert len({float(t) for t in a[0]}) == 4


@pytest.mark.parametrize("precision", ["bf16", "fp32", "int8"])
def test_the_hidden_block_of_a_dense_program(tt, precision):
    """The executor's spins, read in place, are the features; its next sweep comes after them."""
    prog = workloads.gaussian_bernoulli_rbm(256, 512, seed=2, w_std=0.05)
    ex = tt.Executor(None, tt.open_device(None), prog, tt.make_cuda_config(dense_precision=precision), n_chains=128)
    g = torch.Generator().manual_seed(3)
    ex.load_state([torch.randn((128, 256), generator=g), torch.randint(0, 2, (128, 512), generator=g).bool()], [])
    ex._prepare_rng_for_n_sweeps(1, 100)
    r = tt.CategoricalReadout(512, 40, seed=5)
    other = tt.CategoricalReadout(512, 40, seed=5)
    _, y = data(128, 1, 40, 3)
    for _ in range(3):
        ex.run_sweeps(1)
        torch.cuda.synchronize()
        units = ex.dense_units(1).clone()
        assert units.shape == (128, 512) and set(units.float().unique().tolist()) <= {-1.0, 1.0}
        a = r.step(ex, y)
        ex.run_sweeps(1)
        assert torch.equal(a, other.step(units, y))
    torch.cuda.synchronize()
    assert torch.equal(r.weights, other.weights)
    assert torch.equal(r.loss(ex, y), other.loss(ex.dense_units(1), y))
    r.quantize()
    other.quantize()
    assert torch.equal(r.fields(ex), other.fields(ex.dense_units(1).clone()))


def test_units_that_are_still_made_are_waited_for(tt, monkeypatch):
    """Units that are rounded on the executor's stream are used after that, however late it comes."""
    prog = workloads.gaussian_bernoulli_rbm(32, 64, seed=2, w_std=0.05)
    ex = tt.Executor(None, tt.open_device(None), prog, tt.make_cuda_config(dense_precision="fp32"), n_chains=16)
    g = torch.Generator().manual_seed(3)
    spins = torch.randint(0, 2, (16, 64), generator=g).bool()
    ex.load_state([torch.randn((16, 32), generator=g), spins], [])
    units = torch.where(spins, 1.0, -1.0).bfloat16().cuda()
    _, y = data(16, 1, 10, 3)
    r = tt.CategoricalReadout(64, 10, seed=5)
    want = r.loss(units, y)
    torch.cuda.synchronize()

    def late(block):
        with torch.cuda.stream(ex.stream):
            held = torch.zeros_like(units)
            torch.cuda._sleep(200_000_000)
            return held.copy_(units)

    monkeypatch.setattr(ex, "dense_units", late)
    assert torch.equal(r.loss(ex, y), want)


def test_fields_are_those_of_the_rounded_weights(tt):
    r = tt.CategoricalReadout(256, 500, seed=2)
    with pytest.raises(RuntimeError, match="quantize"):
        r.fields(torch.ones(1, 256, device="cuda"))
    r.quantize()
    for rows in (1, 3, 200):
        spins = torch.where(torch.randn(rows, 256, device="cuda") > 0, 1.0, -1.0).bfloat16()
        fields = r.fields(spins)
        exact = spins.double() @ r.served.dequantize().double().t()
        # spins are exact codes up to two roundings of their scale; sums of at most 256 terms; the rounding to bfloat16
        mag = spins.double().abs() @ r.served.dequantize().double().abs().t()
        assert fields.dtype == torch.bfloat16
        assert ((fields.double() - exact).abs() <= (2 * 32 + 8) * 2.0**-24 * mag + 2.0**-8 * (exact.abs() + 1e-4 * mag)).all()


def test_refusals(tt):
    for kw, match in [({"dtype": torch.float32}, "dtype"), ({"dropout": 1.0}, "dropout"), ({"dropout": -0.1}, "dropout")]:
        with pytest.raises(ValueError, match=match):
            tt.CategoricalReadout(8, 5, **kw)
    r = tt.CategoricalReadout(8, 5)
    x, y = torch.ones(4, 8, device="cuda"), torch.zeros(4, dtype=torch.int64, device="cuda")
    for args, match in [((x.int(), y), "floating"), ((x[:, :7], y), "columns"), ((x, y[:3]), "targets"), ((x.cpu(), y), "CUDA"),
                        ((x[:0], y[:0]), "rows"), ((x[0], y[0]), "rows")]:
        with pytest.raises(ValueError, match=match):
            r.step(*args)
