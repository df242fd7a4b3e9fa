"""Learning the couplings of a dense program from its own samples.

The log likelihood of a Boltzmann machine has the gradient <x y>_data -
<x y>_model for a coupling and <x>_data - <x>_model for a bias.  `dense_moments`
takes those differences from the states of executors on the device,
`DenseLearner` closes the loop: sample, moments, AdamW, new operands.
"""

from __future__ import annotations

from . import _native as nat
from .core import Family, make_cuda_config, open_device
from .executor import Executor
from .moments import launch
from .optim import AdamW
from .quantized import check_operator_errors, mark_written, refuse_shared_outputs, refuse_written_grad, require_cuda


def _torch():
    import torch

    return torch


def dense_moments(terms, *, out=None, accumulate: bool = False):
    """sum of scale * (x^T y, sum x, sum y) over (executor, scale) terms of one dense program's shape.

    Returns float32 (pair [n_0, n_1], block 0 [n_0], block 1 [n_1]); `out` is such
    a triple to write, or, with `accumulate`, to add to.  Ordered after the
    executors' sweeps and before their next ones; queued on the current stream.  All executors (a MeshExecutor counts as
    its local shards) must be on one device.
    An in-kernel wait that expires is reported by check_operator_errors()."""
    torch = _torch()
    # a mesh of chains is the sum of its shards
    terms = [(shard, float(s)) for ex, s in terms for shard in getattr(ex, "shards", [ex])]
    if not terms:
        raise ValueError("dense_moments needs at least one executor")
    first = terms[0][0]
    sizes = [[cb.spec.n_nodes for cb in ex.compiled.blocks] for ex, _ in terms]
    if any(s != sizes[0] or ex._tdev != first._tdev for s, (ex, _) in zip(sizes, terms)):
        raise ValueError(f"executors of different programs or devices: blocks of {sizes}")
    dev = first._tdev
    current = torch.cuda.current_stream(dev)
    rows = [r for ex, s in terms for r in ex._dense_phases(s)]
    M, N = sizes[0]
    if out is None:
        if accumulate:
            raise ValueError("accumulate needs out")
        out = tuple(torch.empty(s, dtype=torch.float32, device=dev) for s in ((M, N), (M,), (N,)))
    else:
        for name, t, shape in zip(("out[0]", "out[1]", "out[2]"), out, ((M, N), (M,), (N,)), strict=True):
            require_cuda(name, t, dev)
            if t.dtype != torch.float32 or tuple(t.shape) != shape or not t.is_contiguous():
                raise ValueError(f"{name} must be contiguous float32 of shape {shape}, got {t.dtype} of {tuple(t.shape)}")
            refuse_written_grad(name, t)
        refuse_shared_outputs([(f"out[{i}]", t) for i, t in enumerate(out)])
        mark_written(*out)
    for ex, _ in terms:
        current.wait_stream(ex.stream)
    nat.bind_device(dev.index)
    for at in range(0, len(rows), nat.MAX_PHASES):
        part = rows[at : at + nat.MAX_PHASES]
        phases = (nat.MomentPhase * len(part))()
        for p, (x, x_ld, y, y_ld, s, sx, sy) in zip(phases, part):
            p.x, p.y, p.x_ld, p.y_ld, p.chains = x.data_ptr(), y.data_ptr(), x_ld, y_ld, x.shape[0]
            p.scale, p.x_scale, p.y_scale = s, sx, sy
        launch(phases, nat.DT_BF16, M, N, out[0], out[1], out[2], accumulate or at > 0, dev, current.cuda_stream)
    for ex, _ in terms:
        ex.stream.wait_stream(current)
    return out


class DenseLearner:
    """Persistent contrastive divergence (Tieleman, ICML 2008) of a dense two-block program.

    program: a DenseBipartiteProgram (gaussian or spin visible block 0, spin
    hidden block 1); its couplings and biases are the start.  n_data: rows per
    batch, n_chains: persistent chains of the model (multiples of 128).  config:
    dense_precision "bf16", "fp32" or "int8" for the samplers.  The masters
    `weights` [n_visible, n_hidden], `visible_bias` and `hidden_bias` are float32
    tensors on the device, stepped by `optimizer` (AdamW; `state_bits`).

    step(batch) clamps the visible block of the data chains to the batch, draws
    their hidden units, runs `sweeps` sweeps of the persistent chains, takes the
    moment differences, steps the masters and rounds them into both samplers'
    operands.  It returns the gradient of minus the mean log likelihood as the
    triple that was stepped with (overwritten by the next step).  It does not wait
    for its own work.  A batch in host memory (complete when step is called) has been
    read when step returns, so the caller may fill it anew at once: the copy runs
    beside the device's work, and the host stays within two steps of it.
    check() raises if a kernel of the steps so far gave up a wait: the masters are
    not to be relied on then.
    """

    def __init__(self, program, *, n_data, n_chains, config=None, device=None, sweeps=1, lr=1e-3, betas=(0.9, 0.999),
                 eps=1e-8, weight_decay=0.0, state_bits=32, seed=0):
        torch = _torch()
        config = make_cuda_config() if config is None else config
        if config.rng_mode != "philox":
            raise ValueError("DenseLearner draws on the device: rng_mode must be 'philox'")
        if int(sweeps) < 1:
            raise ValueError(f"sweeps must be at least 1, got {sweeps}")
        if device is None:  # both samplers on one stream
            device = open_device(None, device_id=torch.cuda.current_device())
        self.program, self.sweeps = program, int(sweeps)
        self.data = Executor(None, device, program, config, n_chains=int(n_data))
        self.model = Executor(None, device, program, config, n_chains=int(n_chains))
        plans = self.data._dense_plans("DenseLearner")
        self.model._dense_plans("DenseLearner")
        if plans[1].family != Family.SPIN:
            raise ValueError("DenseLearner needs a spin hidden block (block 1)")
        self._visible_family = plans[0].family
        dev = self.data._tdev
        couplings = program.tt_dense_couplings()
        self.weights = torch.tensor(couplings[0]["weights_nk"], dtype=torch.float32, device=dev)
        self.visible_bias = torch.tensor(couplings[0]["bias"], dtype=torch.float32, device=dev)
        self.hidden_bias = torch.tensor(couplings[1]["bias"], dtype=torch.float32, device=dev)
        self.gradient = tuple(torch.empty_like(t) for t in (self.weights, self.visible_bias, self.hidden_bias))
        self.optimizer = AdamW((self.weights, self.visible_bias, self.hidden_bias), lr=lr, betas=betas, eps=eps,
                               weight_decay=weight_decay, state_bits=state_bits, seed=seed)
        n_v, n_h = self.weights.shape
        g = torch.Generator().manual_seed(int(seed) & 0x7FFFFFFF)

        def start(rows, n, family):
            if family == Family.SPIN:
                return (torch.randint(0, 2, (rows, n), generator=g) * 2 - 1).to(torch.int8)
            return torch.randn((rows, n), generator=g)

        for k, ex in enumerate((self.data, self.model)):
            ex.load_state([start(ex.n_chains, n_v, self._visible_family), start(ex.n_chains, n_h, Family.SPIN)], [])
            # one stream of draws for the whole run, another one for each executor
            ex._prepare_rng_for_n_sweeps((int(seed) << 1) + k, 2**31 - 1)
        self._copies = torch.cuda.Stream(device=dev)
        self._uploads = [(None, torch.cuda.Event()) for _ in range(2)]
        self._hidden_group = next(gr for gr in self.data.compiled.sampling_groups if tuple(gr.block_indices) == (1,))

    def step(self, batch):
        torch = _torch()
        n, n_v = self.data.n_chains, self.weights.shape[0]
        if not isinstance(batch, torch.Tensor) or tuple(batch.shape) != (n, n_v):
            raise ValueError(f"batch must be a tensor of shape {(n, n_v)}, got {getattr(batch, 'shape', type(batch))}")
        with torch.no_grad():  # the states are drawn: nothing of the batch's graph goes on into them
            return self._step(batch.detach())

    def _step(self, batch):
        torch = _torch()
        data, model = self.data, self.model
        n = data.n_chains
        current = torch.cuda.current_stream(data._tdev)
        upload = self._upload(batch) if batch.device.type == "cpu" else None
        if upload is not None:
            batch = upload[0]
        data.stream.wait_stream(current)
        with torch.cuda.stream(data.stream):
            values = batch.to(data._tdev, non_blocking=True)
            if self._visible_family == Family.SPIN:
                values = torch.where(values > 0, 1.0, -1.0)
            data._dense_write_block(0, values)
            if upload is not None:
                upload[1].record(data.stream)
            elif batch.device == data._tdev:
                batch.record_stream(data.stream)
        data._check_ready()
        data._run_sampling_group(self._hidden_group, data._sweep_counter)
        data._sweep_counter += 1
        model.run_sweeps(self.sweeps)
        dense_moments([(data, -1.0 / n), (model, 1.0 / model.n_chains)], out=self.gradient)
        self.optimizer.step(self.gradient)
        data.update_dense_weights(self.weights, self.visible_bias, self.hidden_bias)
        model.share_dense_weights(data)
        return self.gradient

    def _upload(self, batch):
        """(device copy, event to record when it has been read) of a host batch, on a stream of its own: behind the sweeps
        of earlier steps the copy would still read the batch long after step has returned.  Two buffers in turn keep the
        host within two steps of the device."""
        torch = _torch()
        self._uploads.reverse()
        buffer, read = self._uploads[0]
        with torch.cuda.stream(self._copies):
            self._copies.wait_event(read)
            if buffer is None or buffer.dtype != batch.dtype:
                buffer = torch.empty(batch.shape, dtype=batch.dtype, device=self.data._tdev)
                buffer.record_stream(self.data.stream)
                self._uploads[0] = (buffer, read)
            buffer.copy_(batch)  # waits for the copy
        return self._uploads[0]

    def check(self) -> None:
        """Raises if a kernel of the steps so far gave up an in-kernel wait.  Synchronises."""
        self.data.check_device_errors()
        self.model.check_device_errors()
        check_operator_errors(self.data._tdev)


__all__ = ["dense_moments", "DenseLearner"]
