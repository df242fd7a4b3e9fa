"""Operators of a categorical readout over a dense program's units: cases, plain forms and 64-bit values.

Four operators that a user needs next to the sampling and learning of dense programs:

* `softmax_cross_entropy`: minus the log likelihood of categories under softmax(x W^T + b), x the units' values of a
  batch of rows, with the gradients of x, W and b; the logits are never held as a whole.
* `quantize_fp4`: rows as 4-bit floating point values (e2m1) with an 8-bit scale (e4m3) per 16 columns and a float32
  scale per row.
* `fp4_product`: products of such rows (floats are quantised within the call) with such weights.
* `dropout`: elements dropped by bits of a counter-based generator, with the gradient; the mask is not held.

`own` False computes the plain forms (elementary torch operations); True calls tt_thrml_b200.
"""

from __future__ import annotations

import math

import numpy as np
import torch

own = False

DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
BYTES = {"fp32": 4, "bf16": 2, "fp16": 2}
DEVICE = "cuda"

BLOCK = 16  # columns that share a scale of 8 bits
TOP = 6.0 * 448.0  # the largest code times the largest scale of a block
SALT = 0x44524F50  # counter word of the dropout's draws
IGNORED = -100


def listed():
    return [
        # one chain's hidden units (the small test RBM's 512) against a thousand categories: latency of a training step
        {"name": "xent-train-1x512x1000-bf16", "op": "xent", "rows": 1, "k": 512, "v": 1000, "dtype": "bf16",
         "bias": True, "train": True},
        # evaluation of 64 rows over a large vocabulary: the weights are read once
        {"name": "xent-eval-64x4096x32768-bf16", "op": "xent", "rows": 64, "k": 4096, "v": 32768, "dtype": "bf16",
         "bias": False, "train": False},
        # odd sizes everywhere, half precision
        {"name": "xent-train-777x1001x5003-fp16", "op": "xent", "rows": 777, "k": 1001, "v": 5003, "dtype": "fp16",
         "bias": True, "train": True},
        # the visible units of the 4096 x 8192 RBM, a minibatch of 1024 rows, a large ragged vocabulary
        {"name": "xent-train-1024x4096x50021-bf16", "op": "xent", "rows": 1024, "k": 4096, "v": 50021, "dtype": "bf16",
         "bias": True, "train": True},
        # all 8192 chains of that RBM
        {"name": "xent-train-8192x4096x32768-bf16", "op": "xent", "rows": 8192, "k": 4096, "v": 32768, "dtype": "bf16",
         "bias": False, "train": True},
        # odd rows into 4 bits, half precision
        {"name": "fp4-quantize-37x5001-fp16", "op": "quantize", "rows": 37, "k": 5001, "dtype": "fp16"},
        # the 4096 x 8192 RBM's weights into 4 bits
        {"name": "fp4-quantize-8192x4096-bf16", "op": "quantize", "rows": 8192, "k": 4096, "dtype": "bf16"},
        # one chain's hidden fields (a single token): latency
        {"name": "fp4-1x4096x8192-bf16", "op": "fp4", "rows": 1, "k": 4096, "n": 8192, "dtype": "bf16", "bias": True},
        # a handful of rows, odd sizes everywhere, half precision
        {"name": "fp4-37x5001x2047-fp16", "op": "fp4", "rows": 37, "k": 5001, "n": 2047, "dtype": "fp16",
         "bias": False},
        # the RBM's hidden fields of all 8192 chains
        {"name": "fp4-8192x4096x8192-bf16", "op": "fp4", "rows": 8192, "k": 4096, "n": 8192, "dtype": "bf16",
         "bias": True},
        # the small test RBM's hidden units of 64 rows, forward and backward: latency
        {"name": "dropout-64x512-fp32", "op": "dropout", "rows": 64, "k": 512, "dtype": "fp32", "p": 0.5},
        # the hidden units of 8192 chains, forward and backward
        {"name": "dropout-8192x8192-bf16", "op": "dropout", "rows": 8192, "k": 8192, "dtype": "bf16", "p": 0.1},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["xent", "xent", "quantize", "fp4", "dropout"])
    half = rng.choice(["bf16", "fp16"])
    if op == "xent":
        c = {"op": op, "rows": _log(rng, 1, 16384), "k": _log(rng, 8, 8192), "v": _log(rng, 2, 131072), "dtype": half,
             "bias": rng.random() < 0.5, "train": rng.random() < 0.7}
        c["rows"] = max(1, min(c["rows"], 8192 * 4096 * 32768 // (c["k"] * c["v"]), (1 << 29) // c["v"]))
        return c
    if op == "quantize":
        return {"op": op, "rows": _log(rng, 1, 8192), "k": _log(rng, 16, 16384), "dtype": rng.choice(list(DTYPES))}
    if op == "fp4":
        c = {"op": op, "rows": _log(rng, 1, 8192), "k": _log(rng, 16, 8192), "n": _log(rng, 16, 8192), "dtype": half,
             "bias": rng.random() < 0.5}
        c["rows"] = max(1, min(c["rows"], 8192 * 4096 * 8192 // (c["k"] * c["n"])))
        return c
    return {"op": op, "rows": _log(rng, 1, 8192), "k": _log(rng, 1, 8192), "dtype": rng.choice(list(DTYPES)),
            "p": rng.choice([0.1, 0.2, 0.5, 0.9])}


def _held(rows, k):
    """Bytes of rows of 4-bit values with their scales."""
    return rows * ((k + 1) // 2 + (k + BLOCK - 1) // BLOCK + 4)


def work(case):
    b = BYTES[case["dtype"]]
    rows, k = case["rows"], case["k"]
    if case["op"] == "xent":
        v, train = case["v"], case["train"]
        read = b * (rows * k + v * k) + 8 * rows + (4 * v if case["bias"] else 0)
        wrote = b * (rows * k + v * k) + (4 * v if case["bias"] else 0) + 4 if train else 4 * rows
        return {"bytes": read + wrote, "flops": (6 if train else 2) * rows * k * v}
    if case["op"] == "quantize":  # the values that the codes stand for are written out
        return {"bytes": rows * k * (b + 4) + 2 * _held(rows, k), "flops": 8 * rows * k}
    if case["op"] == "fp4":
        n = case["n"]
        return {"bytes": b * rows * (k + n) + _held(n, k) + (4 * n if case["bias"] else 0), "flops": 2 * rows * k * n}
    return {"bytes": 4 * rows * k * b, "flops": 12 * rows * k}


def _inputs(case, seed):
    g = torch.Generator(device=DEVICE)
    g.manual_seed(seed)
    t = DTYPES[case["dtype"]]
    rows, k = case["rows"], case["k"]

    def normal(*shape):
        return torch.randn(shape, generator=g, device=DEVICE)

    if case["op"] == "xent":
        v = case["v"]
        targets = torch.randint(0, v, (rows,), generator=g, device=DEVICE)
        padded = torch.rand(rows, generator=g, device=DEVICE) < 0.05
        if rows > 1:  # some rows of a batch are padding
            targets = torch.where(padded, IGNORED, targets)
        return {"x": normal(rows, k).to(t), "w": (normal(v, k) * (1.5 / math.sqrt(k))).to(t), "targets": targets,
                "bias": normal(v) * 0.5 if case["bias"] else None}
    if case["op"] == "quantize":
        return {"x": (normal(rows, k) * 0.02).to(t)}
    if case["op"] == "fp4":
        n = case["n"]
        blocks = -(-k // BLOCK)
        codes = torch.randint(0, 16, (n, 2 * ((k + 1) // 2)), generator=g, device=DEVICE, dtype=torch.uint8)
        if k % 2:
            codes[:, k] = 0
        # scales of blocks as a row of normal weights has them: most between a third of the largest and the largest
        scale = (448.0 * (0.3 + 0.7 * torch.rand((n, blocks), generator=g, device=DEVICE))).to(torch.float8_e4m3fn)
        return {"x": normal(rows, k).to(t), "w_codes": codes[:, 0::2] | codes[:, 1::2] << 4, "w_block": scale,
                "w_scale": (0.5 + torch.rand(n, generator=g, device=DEVICE)) * (0.04 / TOP),
                "bias": normal(n) * 0.3 if case["bias"] else None}
    return {"x": normal(rows, k).to(t), "grad": normal(rows, k).to(t), "seed": (seed * 0x9E3779B97F4A7C15 + 1) % 2**64,
            "step": seed % 1000}


def prepare(case, seed):
    s = _inputs(case, seed)
    s["case"] = case
    if own:
        import tt_thrml_b200 as tt

        if case["op"] == "fp4":
            s["weights"] = tt.Fp4Rows(s["w_codes"], s["w_block"], s["w_scale"], cols=case["k"])
        elif case["op"] == "dropout" or case.get("train"):
            for name in ("x", "w", "bias"):
                if s.get(name) is not None:
                    s[name].requires_grad_(True)
    return s


def run(s):
    case = s["case"]
    if own:
        import tt_thrml_b200 as tt

        if case["op"] == "xent":
            if not case["train"]:
                return tt.softmax_cross_entropy(s["x"], s["w"], s["targets"], bias=s["bias"], reduction="none")
            loss = tt.softmax_cross_entropy(s["x"], s["w"], s["targets"], bias=s["bias"])
            leaves = [s["x"], s["w"]] + ([] if s["bias"] is None else [s["bias"]])
            return (loss.detach(), *torch.autograd.grad(loss, leaves))
        if case["op"] == "quantize":
            return tt.quantize_fp4(s["x"]).dequantize()
        if case["op"] == "fp4":
            return tt.fp4_product(s["x"], s["weights"], bias=s["bias"])
        y = tt.dropout(s["x"], case["p"], seed=s["seed"], step=s["step"])
        return (y.detach(), *torch.autograd.grad(y, s["x"], s["grad"]))
    if case["op"] == "xent":
        return _xent_plain(s)
    if case["op"] == "quantize":
        q, scale = _fp4_plain(s["x"])
        return q * scale
    return _product_plain(s) if case["op"] == "fp4" else _dropout_plain(s)


def _xent_plain(s):
    """loss = log sum exp l - l[y], l = x W^T + b; with the mean over the rows that count, its gradients."""
    x, w, y = s["x"].float(), s["w"].float(), s["targets"]
    logits = x @ w.t()
    if s["bias"] is not None:
        logits += s["bias"]
    top = logits.amax(1, keepdim=True)
    p = torch.exp(logits - top)
    total = p.sum(1, keepdim=True)
    counts = y != IGNORED
    at = torch.where(counts, y, 0)[:, None]
    loss = torch.where(counts, (torch.log(total) + top - logits.gather(1, at))[:, 0], 0.0)
    if not s["case"]["train"]:
        return loss
    n = counts.sum().clamp(min=1)
    p /= total
    p.scatter_add_(1, at, torch.full_like(top, -1.0))
    p *= (counts / n)[:, None]
    out = (loss.sum() / n, (p @ w).to(s["x"].dtype), (p.t() @ x).to(s["w"].dtype))
    return out if s["bias"] is None else (*out, p.sum(0))


def _blocks(x):
    """Rows cut into blocks of 16 columns, the last one filled with zeros: [rows, blocks, 16]."""
    return torch.nn.functional.pad(x, (0, -x.shape[1] % BLOCK)).unflatten(1, (-1, BLOCK))


def _fp4_plain(x):
    """(code times the block's scale, the row's scale) of the rows of x, decided in float32."""
    f = x.float()
    top = f.abs().amax(1, keepdim=True)
    inv = torch.div(torch.full_like(top, TOP), top)
    b = _blocks(f)
    e = ((b.abs().amax(2) * inv) * (1.0 / 6.0)).clamp(max=448.0).to(torch.float8_e4m3fn).float()
    y = b * torch.where(e > 0, torch.div(inv.expand_as(e), e), 0.0)[:, :, None]
    a = y.abs().clamp(max=6.0)
    step = torch.where(a < 2.0, 0.5, torch.where(a < 4.0, 1.0, 2.0))
    q = torch.copysign(torch.round(a / step) * step, y) * e[:, :, None]
    return q.flatten(1)[:, : x.shape[1]], top * (1.0 / TOP)


def _product_plain(s):
    """y = (sum_k q w) (s_x s_w) + bias, q and w codes times their blocks' scales, rounded once to x's type."""
    k = s["case"]["k"]
    q, scale = _fp4_plain(s["x"])
    packed = s["w_codes"]
    codes = torch.stack([packed & 15, packed >> 4], 2).flatten(1)[:, :k]
    grid = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], device=packed.device)
    w = torch.cat([grid, -grid])[codes.int()]
    w = (_blocks(w) * s["w_block"].float()[:, :, None]).flatten(1)[:, :k]
    y = (q @ w.t()) * (scale * s["w_scale"])
    return (y if s["bias"] is None else y + s["bias"]).to(s["x"].dtype)


def _philox(n, seed, step):
    """Philox4x32-10 on counters (i, i >> 32, step, SALT), i < n: int64 [n, 4] of 32-bit values."""
    low = 0xFFFFFFFF
    i = torch.arange(n, device=DEVICE, dtype=torch.int64)
    x, y = i & low, i >> 32
    z, w = torch.full_like(i, step & low), torch.full_like(i, SALT)
    k0, k1 = seed & low, seed >> 32
    for _ in range(10):
        a, b = x * 0xD2511F53, z * 0xCD9E8D57
        x, y, z, w = ((b >> 32) & low) ^ y ^ k0, b & low, ((a >> 32) & low) ^ w ^ k1, a & low
        k0, k1 = (k0 + 0x9E3779B9) & low, (k1 + 0xBB67AE85) & low
    return torch.stack([x, y, z, w], 1)


def _dropout_plain(s):
    """Element i is kept where half-word i % 8 of draw i // 8 is at least round(65536 p), and scaled to keep its mean."""
    x, n = s["x"], s["x"].numel()
    words = _philox((n + 7) // 8, s["seed"], s["step"])
    bits = torch.stack([words & 0xFFFF, words >> 16], 2).flatten()[:n].view_as(x)
    cut = round(65536 * s["case"]["p"])
    scale = 65536.0 / (65536.0 - cut)
    return tuple(torch.where(bits >= cut, t.float() * scale, 0.0).to(t.dtype) for t in (x, s["grad"]))


def _fp4_exact(x):
    """Codes times the blocks' scales, which are float32 decisions by definition, and the rows' scales in 64 bits."""
    f = x.float()
    top = f.abs().max(1).values
    inv = torch.full_like(top, TOP) / top
    pad = torch.zeros((x.shape[0], -(-x.shape[1] // BLOCK) * BLOCK), device=x.device)
    pad[:, : x.shape[1]] = f
    b = pad.view(x.shape[0], -1, BLOCK)
    t = (b.abs().max(2).values * inv[:, None] * (1.0 / 6.0)).double()
    # e4m3: three bits below the leading one, none below 2^-9
    unit = torch.exp2(torch.floor(torch.log2(t.clamp(min=2.0**-6))) - 3.0)
    e = (torch.round(t / unit) * unit).clamp(max=448.0)
    y = b * torch.where(e > 0, inv[:, None].expand_as(e) / e.float(), torch.zeros_like(inv)[:, None])[:, :, None]
    a = y.abs().double()
    # the places where a larger code begins: a tie goes to the even one of its two neighbours
    value = sum(gap * (a > at if even else a >= at)
                for at, gap, even in ((0.25, 0.5, True), (0.75, 0.5, False), (1.25, 0.5, True), (1.75, 0.5, False),
                                      (2.5, 1.0, True), (3.5, 1.0, False), (5.0, 2.0, True)))
    q = value * torch.sign(y).double() * e[:, :, None]
    return q.reshape(x.shape[0], -1)[:, : x.shape[1]], top.double() / TOP


def exact(case, seed):
    s = _inputs(case, seed)
    if case["op"] == "xent":
        x, w, y = s["x"].double(), s["w"].double(), s["targets"]
        logits = torch.einsum("tk,vk->tv", x, w)
        if s["bias"] is not None:
            logits = logits + s["bias"].double()[None, :]
        log_p = logits - torch.logsumexp(logits, 1)[:, None]
        rows = torch.arange(case["rows"], device=DEVICE)
        live = (y != IGNORED).double()
        y = y.clamp(min=0)
        loss = -log_p[rows, y] * live
        if not case["train"]:
            return loss
        weight = live / max(1.0, float(live.sum()))
        g = torch.exp(log_p)
        g[rows, y] -= 1.0
        g = weight[:, None] * g
        out = ((loss * weight).sum(), torch.einsum("tv,vk->tk", g, w), torch.einsum("tv,tk->vk", g, x))
        return out if s["bias"] is None else (*out, torch.einsum("tv->v", g))
    if case["op"] == "quantize":
        q, scale = _fp4_exact(s["x"])
        return q * scale[:, None]
    if case["op"] == "fp4":
        q, scale = _fp4_exact(s["x"])
        high, low = s["w_codes"].int() // 16, s["w_codes"].int() % 16
        c = torch.empty((case["n"], 2 * high.shape[1]), dtype=torch.float64, device=DEVICE)
        for at, code in ((0, low), (1, high)):
            m, power = code % 2, code // 2 % 4  # one bit below the leading one, whose place the next two bits give
            value = torch.where(power > 0, (1.0 + 0.5 * m) * torch.exp2(power - 1.0), 0.5 * m)
            c[:, at::2] = torch.where(code >= 8, -value, value)
        w = c[:, : case["k"]] * s["w_block"].double().repeat_interleave(BLOCK, 1)[:, : case["k"]]
        y = torch.einsum("mk,nk->mn", q, w) * torch.outer(scale, s["w_scale"].double())
        return y if s["bias"] is None else y + s["bias"].double()[None, :]
    keep, scale = _kept(case["rows"] * case["k"], s["seed"], s["step"], case["p"])
    return tuple(t.double() * keep.view_as(t) * scale for t in (s["x"], s["grad"]))


def _kept(n, seed, step, p):
    """Which of n elements the dropout keeps, from the generator in 64-bit host arithmetic, and their factor."""
    i = np.arange((n + 7) // 8, dtype=np.uint64)
    low, c32 = np.uint64(0xFFFFFFFF), np.uint64(32)
    c = [i & low, i >> c32, np.full_like(i, step), np.full_like(i, SALT)]
    key = [seed % 2**32, seed // 2**32]
    for _ in range(10):
        a, b = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        c = [b >> c32 ^ c[1] ^ np.uint64(key[0]), b & low, a >> c32 ^ c[3] ^ np.uint64(key[1]), a & low]
        key = [(key[0] + 0x9E3779B9) % 2**32, (key[1] + 0xBB67AE85) % 2**32]
    cut = round(p * 65536)
    half = np.stack([part for word in c for part in (word & np.uint64(0xFFFF), word >> np.uint64(16))], 1)
    keep = torch.from_numpy((half.reshape(-1)[:n] >= cut).astype(np.float64))
    return keep.to(DEVICE), 1.0 / (1.0 - cut / 65536)
