"""Categories read out of a block's units.

    p(v | x) = softmax(x W^T + b)_v

x is the hidden block of a dense program over its chains (or any features), v one
of many categories: labels of the data, or the words of a vocabulary.
`CategoricalReadout` learns W and b from pairs of units and categories: dropout of
the units, softmax cross entropy, AdamW.  What it has learned it serves from 4-bit
weights.
"""

from __future__ import annotations

from .executor import Executor
from .fp4 import fp4_product, quantize_fp4
from .losses import mean_and_gradients, softmax_cross_entropy
from .optim import AdamW
from .quantized import check_operator_errors, require_cuda
from .regularise import dropout as drop


def _torch():
    import torch

    return torch


class CategoricalReadout:
    """softmax(x W^T + b) over n_categories of n_units features.

    dtype: bfloat16 or float16, the type of the products' operands.  dropout: the
    probability with which `step` leaves out a unit.  The masters `weights`
    [n_categories, n_units] (normal of variance 1 / n_units) and `bias` (zeros) are
    float32 tensors on the device, stepped by `optimizer` (AdamW; `state_bits`).

    step(x, targets) takes a step and returns the mean loss before it, a float32
    scalar on the device; its gradients are `gradient` (weights, bias), overwritten by
    the next step.  x: [rows, n_units], or an Executor of a dense program whose hidden block
    (block 1) has n_units, a row per chain.  targets: int64 or int32 [rows],
    `ignore_index` for rows that do not count.  Nothing waits for the device; a step
    on a tensor may be captured into a CUDA graph after a first one outside, and
    leaves out other units each time the graph is replayed.
    loss(x, targets): the mean loss without dropout.
    quantize() rounds the weights to 4 bits (`served`) and keeps the bias that goes with
    them; fields(x) are then x W^T + b of both, in x's type, whatever steps come after.
    check() raises if a kernel gave up an in-kernel wait.
    """

    def __init__(self, n_units, n_categories, *, dtype=None, dropout=0.0, lr=1e-3, betas=(0.9, 0.999), eps=1e-8,
                 weight_decay=0.0, state_bits=32, seed=0, ignore_index=-100, device=None):
        torch = _torch()
        dtype = torch.bfloat16 if dtype is None else dtype
        if dtype not in (torch.bfloat16, torch.float16):
            raise ValueError(f"dtype must be bfloat16 or float16, got {dtype}")
        if not 0.0 <= float(dropout) < 1.0:
            raise ValueError(f"dropout must be at least 0 and below 1, got {dropout}")
        dev = torch.device("cuda", torch.cuda.current_device()) if device is None else torch.device(device)
        g = torch.Generator().manual_seed(int(seed) & 0x7FFFFFFF)
        shape = (int(n_categories), int(n_units))
        self.weights = (torch.randn(shape, generator=g, dtype=torch.float32) * shape[1] ** -0.5).to(dev)
        self.bias = torch.zeros(shape[0], dtype=torch.float32, device=dev)
        self.dropout, self.seed, self.ignore_index = float(dropout), int(seed) & (2**64 - 1), int(ignore_index)
        self.optimizer = AdamW((self.weights, self.bias), lr=lr, betas=betas, eps=eps, weight_decay=weight_decay,
                               state_bits=state_bits, seed=seed)
        self.gradient = (torch.empty_like(self.weights), torch.empty_like(self.bias))
        self._operands = self.weights.to(dtype)
        self._steps = torch.zeros(1, dtype=torch.int64, device=dev)  # which mask of the seed's
        self._one = torch.ones((), dtype=torch.float32, device=dev)
        self.served = self._served_bias = None

    @property
    def device(self):
        return self.weights.device

    def _units(self, x):
        """(the features in the operands' type, the executor that is to wait for their use or None)."""
        torch = _torch()
        if isinstance(x, Executor):
            units = x.dense_units(1)  # float32 states are rounded on the executor's stream, so that stream is waited for after
            torch.cuda.current_stream(self.device).wait_stream(x.stream)
            return units.to(self._operands.dtype), x
        require_cuda("x", x, self.device)
        if not x.is_floating_point():
            raise ValueError(f"x must hold floating point units, got {x.dtype}")
        return x.detach().to(self._operands.dtype), None

    def _used(self, source) -> None:
        if source is not None:
            source.stream.wait_stream(_torch().cuda.current_stream(self.device))

    def step(self, x, targets):
        torch = _torch()
        with torch.no_grad():
            units, source = self._units(x)
            if self.dropout:
                units = drop(units, self.dropout, seed=self.seed, step=self._steps)
            loss = mean_and_gradients(units, self._operands, targets, self.bias, self.ignore_index, self._one, *self.gradient)
            if self.dropout:
                self._steps += 1  # a step that was refused takes no mask
            self._used(source)
            self.optimizer.step(self.gradient)
            self._operands.copy_(self.weights)
        return loss

    def loss(self, x, targets):
        with _torch().no_grad():
            units, source = self._units(x)
            loss = softmax_cross_entropy(units, self._operands, targets, bias=self.bias, ignore_index=self.ignore_index)
            self._used(source)
        return loss

    def quantize(self) -> None:
        self.served, self._served_bias = quantize_fp4(self.weights), self.bias.clone()

    def fields(self, x):
        if self.served is None:
            raise RuntimeError("quantize() makes the weights that fields are served from")
        if not isinstance(x, Executor):
            return fp4_product(x, self.served, bias=self._served_bias)
        with _torch().no_grad():
            units, source = self._units(x)
            fields = fp4_product(units, self.served, bias=self._served_bias)
            self._used(source)
        return fields

    def check(self) -> None:
        """Raises if a kernel of the calls so far gave up an in-kernel wait.  Synchronises."""
        check_operator_errors(self.device)


__all__ = ["CategoricalReadout"]
