"""AdamW over many tensors in one launch, moments in float32 or in 8-bit codes.

    m = b1 m + (1 - b1) g          v = b2 v + (1 - b2) g^2
    p = p (1 - lr wd) - (lr / (1 - b1^t)) m / (sqrt(v) / sqrt(1 - b2^t) + eps)

in float32 throughout: a v that float32 cannot hold (below 7e-46) is 0, as it is in float32 arithmetic elsewhere.

What a sampler's moments are turned into: the couplings and biases of a
program (see `pair_moments` and `DenseLearner`) are tensors of very different
sizes, stepped together.  With `state_bits=8` the moments take 2 bytes and a
32nd instead of 8 per element; the codes are rounded at random with the mean
kept, from a counter-based generator, so a run can be repeated.

The step counter and the learning rate live on the device: a step captured
into a CUDA graph counts on at every replay, and setting `lr` reaches replayed
graphs.  Nothing synchronises.
"""

from __future__ import annotations

import ctypes

import numpy as np

from . import _native as nat
from .quantized import current_device, dtype_code, on_device, raw_stream, require_cuda

BLOCK = 256  # elements per scale of 8-bit moments; segments of the moments are padded to it


def _torch():
    import torch

    return torch


def _dense_order(t):
    """The order of a tensor's elements in memory as (sizes, strides) of its dimensions longer than one,
    outermost first, or None if it has gaps or overlaps."""
    if not t.numel():
        return ()
    dims = sorted(((st, s) for s, st in zip(t.shape, t.stride()) if s != 1), reverse=True)
    want = 1
    for st, s in reversed(dims):
        if st != want:
            return None
        want *= s
    return tuple(st if s != 1 else 0 for s, st in zip(t.shape, t.stride()))


class AdamW:
    """AdamW bound to a list of parameter tensors on one CUDA device.

    params: float32, bfloat16 or float16 tensors without gaps or overlaps
    (any order of dimensions).  `step(grads)` takes one gradient per parameter:
    the parameter's type or float32, the parameter's shape and memory order;
    None reads every parameter's `.grad`.  16-bit parameters are rounded to
    nearest after the step.  state_bits: 32, or 8 for coded moments
    (`seed` keys their rounding).  Of the settings `lr` alone may be changed later.
    A gradient may be its parameter's own memory, but no other parameter's.
    """

    def __init__(self, params, *, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.01, state_bits=32, seed=0):
        torch = _torch()
        self.params = list(params)
        if not self.params:
            raise ValueError("AdamW needs at least one parameter")
        dev = getattr(self.params[0], "device", None)
        for i, p in enumerate(self.params):
            if not (isinstance(p, torch.Tensor) and p.is_cuda and p.device == dev):
                require_cuda(f"parameter {i}", p, dev)
            if dtype_code(p.dtype) is None:
                raise ValueError(f"parameter {i} must be float32, bfloat16 or float16, got {p.dtype}")
            if not p.is_contiguous() and _dense_order(p) is None:
                raise ValueError(f"parameter {i} has gaps or overlaps in memory (strides {tuple(p.stride())})")
        spans = sorted((p.data_ptr(), p.data_ptr() + p.numel() * p.element_size(), i)
                       for i, p in enumerate(self.params) if p.numel())
        for (_, end, i), (start, _, j) in zip(spans, spans[1:]):
            if start < end:
                raise ValueError(f"parameters {i} and {j} share memory")
        if state_bits not in (8, 32):
            raise ValueError(f"state_bits must be 8 or 32, got {state_bits!r}")
        if not (0.0 <= betas[0] < 1.0 and 0.0 <= betas[1] < 1.0):
            raise ValueError(f"betas must lie in [0, 1), got {betas!r}")
        if not eps >= 1e-30 or not weight_decay >= 0.0 or not lr >= 0.0:
            raise ValueError("eps must be at least 1e-30, lr and weight_decay not below 0")
        self.device, self._betas, self._eps, self._weight_decay = dev, tuple(map(float, betas)), float(eps), float(weight_decay)
        self._state_bits, self._seed = int(state_bits), int(seed) & 0xFFFFFFFFFFFFFFFF
        # segment of each parameter in the moments
        self.offsets, total = [], 0
        for p in self.params:
            self.offsets.append(total)
            total += -(-p.numel() // BLOCK) * BLOCK
        self.elements = total
        kinds = (torch.float32, torch.float32) if state_bits == 32 else (torch.int8, torch.uint8)
        self.exp_avg, self.exp_avg_sq = (torch.zeros(max(total, BLOCK), dtype=k, device=dev) for k in kinds)
        self.exp_avg_scale = self.exp_avg_sq_scale = None
        if state_bits == 8:
            self.exp_avg_scale, self.exp_avg_sq_scale = (
                torch.zeros(max(total, BLOCK) // BLOCK, dtype=torch.float32, device=dev) for _ in range(2)
            )
        self._ctl = torch.zeros(3, dtype=torch.int64, device=dev)  # tthrml_adamw_ctl: step, lr (float64), ticket
        self._lr, self._lr_captured = None, False
        self.lr = lr
        self._kinds = [(p.dtype, p.device, p.shape, p.stride()) for p in self.params]
        # tthrml_adamw_tensor rows of the parameters that have elements
        self._live = [i for i, p in enumerate(self.params) if p.numel()]
        self._rows = np.zeros(len(self._live), dtype=np.dtype(nat.AdamWTensor))
        for name, values in (("n", [p.numel() for p in self.params]), ("state", self.offsets),
                             ("param", [p.data_ptr() for p in self.params]),
                             ("param_dtype", [dtype_code(p.dtype) for p in self.params])):
            self._rows[name] = [values[i] for i in self._live]
        self._host = nat.hostcall()
        at = [None if t is None else t.data_ptr() for t in
              (self.exp_avg, self.exp_avg_sq, self.exp_avg_scale, self.exp_avg_sq_scale, self._ctl)]
        self._call = nat.AdamWCall(self._rows.ctypes.data, len(self._rows), self.state_bits, *at, *self.betas, self.eps,
                                   self.weight_decay, self.seed)
        self._call_at, self._entry = ctypes.addressof(self._call), nat.address_of("tthrml_adamw_step")
        self._values_entry = nat.address_of("tthrml_adamw_values")

    # ---------------------------------------------------------------- control

    # fixed when the optimizer is made: captured steps and the host module's calls hold them
    betas = property(lambda self: self._betas)
    eps = property(lambda self: self._eps)
    weight_decay = property(lambda self: self._weight_decay)
    state_bits = property(lambda self: self._state_bits)
    seed = property(lambda self: self._seed)

    @property
    def lr(self) -> float:
        return self._lr

    @lr.setter
    def lr(self, value) -> None:
        """Queued on the current stream; steps launched (or replayed) after it use the new rate.  In a capture it becomes
        part of the graph: every replay sets the rate anew."""
        value = float(value)
        if not value >= 0.0:
            raise ValueError(f"lr must not be below 0, got {value}")
        torch = _torch()
        with torch.cuda.device(self.device):
            # a captured setting acts when it is replayed, which the host does not see: from then on none is skipped
            self._lr_captured = self._lr_captured or torch.cuda.is_current_stream_capturing()
            if value != self._lr or self._lr_captured:
                self._ctl.view(torch.float64)[1].fill_(value)
        self._lr = value

    @property
    def steps(self) -> int:
        """Steps done (reads the device counter: synchronises)."""
        return int(self._ctl[0].item())

    # ------------------------------------------------------------------- step

    def _check(self, grads) -> None:
        """Fills the rows tensor by tensor; raises unless every gradient has its parameter's device, shape and memory
        order and a fitting type."""
        torch = _torch()
        for i, (p, g, kind) in enumerate(zip(self.params, grads, self._kinds)):
            if g is None:
                raise ValueError(f"parameter {i} has no gradient")
            require_cuda(f"gradient {i}", g, self.device)
            if (p.dtype, p.device, p.shape, p.stride()) != kind:
                raise ValueError(f"parameter {i} changed its type or layout since the optimizer was made")
            if g.dtype not in (p.dtype, torch.float32):
                raise ValueError(f"gradient {i} must be {p.dtype} or float32, got {g.dtype}")
            if g.shape != p.shape or _dense_order(g) != _dense_order(p):
                raise ValueError(
                    f"gradient {i} needs the parameter's shape and memory order: shape {tuple(g.shape)}, strides "
                    f"{tuple(g.stride())} for {tuple(p.shape)}, {tuple(p.stride())}"
                )
        for row, i in zip(self._rows, self._live):
            row["param"], row["grad"] = self.params[i].data_ptr(), grads[i].data_ptr()
            row["grad_dtype"] = dtype_code(grads[i].dtype)

    def step(self, grads=None) -> None:
        """One step of all parameters, queued on the current stream of their device."""
        grads = [p.grad for p in self.params] if grads is None else list(grads)
        if len(self.params) != len(self._kinds):
            raise ValueError(f"made for {len(self._kinds)} parameters, params has {len(self.params)} now")
        if len(grads) != len(self.params):
            raise ValueError(f"{len(self.params)} parameters, {len(grads)} gradients")
        index = self.device.index
        if current_device() == index:
            nat.bind_device(index)
            done = self._host.adamw_step(self.params, grads, self._call_at, self._entry, raw_stream(index), index)
            if done == -1:
                return
            if done < -1:
                nat.check(done + 1000, "tthrml_adamw_step")
        self._check(grads)
        c = self._call
        with on_device(self.device):
            nat.check(
                nat.lib().tthrml_adamw_step(
                    c.rows, c.n_rows, c.state_bits, c.exp_avg, c.exp_avg_sq, c.exp_avg_scale, c.exp_avg_sq_scale, c.ctl,
                    c.beta1, c.beta2, c.eps, c.weight_decay, c.seed, raw_stream(index),
                ),
                "tthrml_adamw_step",
            )
        self._host.bump_versions(self.params)

    # ------------------------------------------------------------------ state

    def state_values(self, flat: bool = False):
        """(first, second) moments as float32: one tensor per parameter in its shape and memory order, or the
        two padded buffers (`flat`).  32-bit moments are returned as the optimizer's own buffers."""
        torch = _torch()
        m, v = self.exp_avg, self.exp_avg_sq
        if self.state_bits == 8:
            index = self.device.index
            with on_device(self.device):
                made = self._host.adamw_values(self._call_at, m, m.numel(), self._values_entry, raw_stream(index))
            if type(made) is int:
                nat.check(made, "tthrml_adamw_values")
            m, v = made
        if flat:
            return (m, v) if m.numel() == self.elements else (m[: self.elements], v[: self.elements])
        return tuple([torch.as_strided(t, p.shape, p.stride(), o) if p.numel() else t[:0].view(p.shape)
                      for p, o in zip(self.params, self.offsets)] for t in (m, v))

    def state_dict(self) -> dict:
        """The state as it is held: step, and copies of the padded buffers (codes and scales with 8 bits)."""
        n = self.elements
        d = {"step": self.steps, "exp_avg": self.exp_avg[:n].clone(), "exp_avg_sq": self.exp_avg_sq[:n].clone()}
        if self.state_bits == 8:
            d |= {"exp_avg_scale": self.exp_avg_scale[: n // BLOCK].clone(),
                  "exp_avg_sq_scale": self.exp_avg_sq_scale[: n // BLOCK].clone()}
        return d

    def load_state_dict(self, state: dict) -> None:
        names = ["exp_avg", "exp_avg_sq"] + (["exp_avg_scale", "exp_avg_sq_scale"] if self.state_bits == 8 else [])
        missing = [k for k in ["step", *names] if k not in state]
        if missing:
            raise ValueError(f"state without {', '.join(missing)}")
        if int(state["step"]) < 0:
            raise ValueError(f"step must not be below 0, got {state['step']}")
        for k in names:
            mine, t = getattr(self, k), state[k]
            n = self.elements // (BLOCK if k.endswith("scale") else 1)
            if tuple(t.shape) != (n,) or t.dtype != mine.dtype:
                raise ValueError(f"{k} must be {mine.dtype} of {n} elements, got {t.dtype} of {tuple(t.shape)}")
        for k in names:
            getattr(self, k)[: state[k].numel()].copy_(state[k])
        self._ctl[0].fill_(int(state["step"]))


__all__ = ["AdamW"]
