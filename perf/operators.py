"""Operators around a dense (restricted Boltzmann) program: cases, plain forms and 64-bit values.

Three operators that a user needs next to the block-Gibbs sweeps of a dense bipartite program:

* `int8_product`: fields of a batch of rows through weights held as 8-bit integers, one scale per row
  (token / chain) and one per output channel (unit); the rows are quantised within the call.
* `pair_moments`: sum over chains of x[c, i] y[c, j] over one or several phases, with the unit sums: the gradient
  of a dense program's couplings and biases (data phase minus model phase).
* `AdamW`: one step of decoupled-weight-decay Adam over many tensors at once, moments in 32 bits or in 8-bit codes.

`own` False computes the plain forms (elementary torch operations); True calls tt_thrml_b200.
"""

from __future__ import annotations

import math
import random

import torch

own = False

DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
BYTES = {"fp32": 4, "bf16": 2, "fp16": 2}
DEVICE = "cuda"

# AdamW: moment codes live in blocks of 256 elements with one scale; a tensor's segment of the flat state is
# padded to whole blocks
BLOCK = 256
LR, BETA1, BETA2, EPS, DECAY = 2e-3, 0.9, 0.999, 1e-8, 0.01
SEED = 0x5EED0123456789AB
SALT = 0x41444D57


def listed():
    return [
        # one chain's hidden fields (a single token): latency
        {"name": "int8-1x4096x8192-bf16", "op": "int8", "rows": 1, "k": 4096, "n": 8192, "dtype": "bf16", "bias": True},
        # a handful of rows, odd sizes everywhere, half precision
        {"name": "int8-37x5001x2047-fp16", "op": "int8", "rows": 37, "k": 5001, "n": 2047, "dtype": "fp16",
         "bias": False},
        # 256 chains, float32 rows in and out
        {"name": "int8-256x8192x4096-fp32", "op": "int8", "rows": 256, "k": 8192, "n": 4096, "dtype": "fp32",
         "bias": True},
        # the 4096 x 8192 RBM: hidden fields of all 8192 chains
        {"name": "int8-8192x4096x8192-bf16", "op": "int8", "rows": 8192, "k": 4096, "n": 8192, "dtype": "bf16",
         "bias": True},
        # the small test RBM (256 x 512), 64 data rows against 128 chains: latency
        {"name": "moments-256x512-64+128", "op": "moments", "x": 256, "y": 512, "data": 64, "model": 128,
         "dtype": "bf16"},
        # ragged: odd unit counts and odd batches
        {"name": "moments-777x1999-500+1023", "op": "moments", "x": 777, "y": 1999, "data": 500, "model": 1023,
         "dtype": "fp16"},
        # the 4096 x 8192 RBM, a minibatch of 1024 rows against 8192 chains
        {"name": "moments-4096x8192-1024+8192", "op": "moments", "x": 4096, "y": 8192, "data": 1024, "model": 8192,
         "dtype": "bf16"},
        # the small test RBM's weights and biases: latency
        {"name": "adamw32-rbm-256x512", "op": "adamw", "layout": "rbm", "x": 256, "y": 512, "bits": 32,
         "dtype": "fp32", "grad": "fp32"},
        # a program of many factors: 600 tensors of 1 to 65536 weights in half precision, 8-bit moments
        {"name": "adamw8-600-bf16", "op": "adamw", "layout": "many", "x": 600, "y": 65536, "bits": 8,
         "dtype": "bf16", "grad": "bf16"},
        # the same tensors with 32-bit moments
        {"name": "adamw32-600-bf16", "op": "adamw", "layout": "many", "x": 600, "y": 65536, "bits": 32,
         "dtype": "bf16", "grad": "bf16"},
        # the 4096 x 8192 RBM's float32 weights and biases, both widths of the moments
        {"name": "adamw32-rbm-4096x8192", "op": "adamw", "layout": "rbm", "x": 4096, "y": 8192, "bits": 32,
         "dtype": "fp32", "grad": "fp32"},
        {"name": "adamw8-rbm-4096x8192", "op": "adamw", "layout": "rbm", "x": 4096, "y": 8192, "bits": 8,
         "dtype": "fp32", "grad": "fp32"},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["int8", "moments", "adamw"])
    if op == "int8":
        c = {"op": op, "rows": _log(rng, 1, 8192), "k": _log(rng, 16, 8192), "n": _log(rng, 16, 8192),
             "dtype": rng.choice(list(DTYPES)), "bias": rng.random() < 0.5}
        c["rows"] = max(1, min(c["rows"], 8192 * 4096 * 8192 // (c["k"] * c["n"])))
        return c
    if op == "moments":
        c = {"op": op, "x": _log(rng, 1, 8192), "y": _log(rng, 1, 8192), "data": _log(rng, 1, 4096),
             "model": _log(rng, 1, 8192), "dtype": rng.choice(["bf16", "fp16"])}
        c["model"] = max(1, min(c["model"], 9216 * 4096 * 8192 // (c["x"] * c["y"]) - c["data"]))
        return c
    dtype = rng.choice(list(DTYPES))
    c = {"op": op, "layout": rng.choice(["rbm", "many"]), "bits": rng.choice([8, 32]), "dtype": dtype,
         "grad": rng.choice([dtype, "fp32"])}
    if c["layout"] == "rbm":
        return c | {"x": _log(rng, 1, 4096), "y": _log(rng, 1, 8192)}
    return c | {"x": _log(rng, 1, 1200), "y": _log(rng, 1, 65536)}


def _sizes(case):
    """Element counts of the tensors of an AdamW case."""
    if case["layout"] == "rbm":
        return [case["x"] * case["y"], case["x"], case["y"]]
    r = random.Random(case["x"] * 1000003 + case["y"])
    return [_log(r, 1, case["y"]) for _ in range(case["x"])]


def work(case):
    if case["op"] == "int8":
        m, k, n, b = case["rows"], case["k"], case["n"], BYTES[case["dtype"]]
        return {"bytes": m * k * b + n * k + 4 * n * (2 if case["bias"] else 1) + m * n * b, "flops": 2 * m * n * k}
    if case["op"] == "moments":
        x, y, c = case["x"], case["y"], case["data"] + case["model"]
        return {"bytes": 2 * c * (x + y) + 4 * (x * y + x + y), "flops": 2 * c * x * y}
    n, p, g = sum(_sizes(case)), BYTES[case["dtype"]], BYTES[case["grad"]]
    if case["bits"] == 32:
        return {"bytes": n * (2 * p + g + 16), "flops": 14 * n}
    # codes read and written with a scale per 256, and the values that the new codes stand for written out
    return {"bytes": n * (2 * p + g + 4 + 8) + n // 16, "flops": 60 * n}


def _generator(seed):
    g = torch.Generator(device=DEVICE)
    g.manual_seed(seed)
    return g


def _inputs(case, seed):
    g = _generator(seed)
    t = DTYPES[case["dtype"]]

    def normal(*shape):
        return torch.randn(shape, generator=g, device=DEVICE)

    def spins(*shape):
        return torch.randint(0, 2, shape, generator=g, device=DEVICE, dtype=torch.int8) * 2 - 1

    if case["op"] == "int8":
        m, k, n = case["rows"], case["k"], case["n"]
        w = normal(n, k) * 0.01
        top = w.abs().amax(1)
        return {"x": normal(m, k).to(t), "w": torch.round(w * (127.0 / top)[:, None]).to(torch.int8),
                "w_scale": top * (1.0 / 127.0), "bias": normal(n) * 0.3 if case["bias"] else None}
    if case["op"] == "moments":
        # gaussian visible units against spins, both phases
        return {"x": [normal(case[p], case["x"]).to(t) for p in ("data", "model")],
                "y": [spins(case[p], case["y"]).to(t) for p in ("data", "model")],
                "scale": [-1.0 / case["data"], 1.0 / case["model"]]}
    sizes = _sizes(case)
    padded = [-(-n // BLOCK) * BLOCK for n in sizes]
    starts, total = [], 0
    for n in padded:
        starts.append(total)
        total += n
    # values and gradients of the tensors lie in one padded buffer each; the padding holds zeros
    live = torch.zeros(total, dtype=torch.bool, device=DEVICE)
    ends = torch.zeros(total + 1, dtype=torch.int32, device=DEVICE)
    at = torch.tensor([starts, [s + n for s, n in zip(starts, sizes)]], device=DEVICE)
    ends.index_add_(0, at[0], torch.ones_like(at[0], dtype=torch.int32))
    ends.index_add_(0, at[1], torch.full_like(at[1], -1, dtype=torch.int32))
    live = torch.cumsum(ends[:-1], 0) > 0
    p = torch.where(live, normal(total) * 0.01, 0.0).to(t)
    grad = torch.where(live, normal(total) * 0.05, 0.0).to(DTYPES[case["grad"]])
    s = {"p": p, "grad": grad, "sizes": sizes, "starts": starts, "step": 100}
    if case["bits"] == 32:
        s["m"] = torch.where(live, normal(total) * 0.015, 0.0)
        s["v"] = torch.where(live, (normal(total) * 0.05).square() + 1e-6, 0.0)
    else:
        s["m"] = torch.where(live, torch.randint(-127, 128, (total,), generator=g, device=DEVICE), 0).to(torch.int8)
        s["v"] = torch.where(live, torch.randint(1, 256, (total,), generator=g, device=DEVICE), 0).to(torch.uint8)
        s["m_scale"] = torch.rand(total // BLOCK, generator=g, device=DEVICE) * 0.02 + 0.01
        s["v_scale"] = torch.rand(total // BLOCK, generator=g, device=DEVICE) * 4e-3 + 2e-3
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    s["case"] = case
    if own:
        import tt_thrml_b200 as tt

        if case["op"] == "int8":
            s["weights"] = tt.QuantizedRows(s["w"], s["w_scale"])
        elif case["op"] == "adamw":
            cut = [slice(a, a + n) for a, n in zip(s["starts"], s["sizes"])]
            s["params"], s["grads"] = [s["p"][c] for c in cut], [s["grad"][c] for c in cut]
            s["opt"] = tt.AdamW(s["params"], lr=LR, betas=(BETA1, BETA2), eps=EPS, weight_decay=DECAY,
                                state_bits=case["bits"], seed=SEED)
            state = {"step": s["step"], "exp_avg": s["m"], "exp_avg_sq": s["v"]}
            if case["bits"] == 8:
                state |= {"exp_avg_scale": s["m_scale"], "exp_avg_sq_scale": s["v_scale"]}
            s["opt"].load_state_dict(state)
    return s


def run(s):
    case = s["case"]
    if own:
        import tt_thrml_b200 as tt

        if case["op"] == "int8":
            return tt.int8_product(s["x"], s["weights"], bias=s["bias"])
        if case["op"] == "moments":
            return tt.pair_moments(s["x"], s["y"], s["scale"], units=True)
        s["opt"].step(s["grads"])
        m, v = s["opt"].state_values(flat=True)
        return {"p": s["p"], "exp_avg": m, "exp_avg_sq": v}
    if case["op"] == "int8":
        return _int8_plain(s)
    return _moments_plain(s) if case["op"] == "moments" else _adamw_plain(s)


def _int8_plain(s):
    """q = round(x 127 / max|x|) per row; y = (q w^T) (s_x s_w) + bias, rounded once to x's type."""
    x = s["x"].float()
    top = x.abs().amax(1, keepdim=True)
    inv = torch.div(torch.full_like(top, 127.0), top)
    q = torch.round(x * inv).clamp(-127.0, 127.0)
    acc = q @ s["w"].float().t()
    y = acc * ((top * (1.0 / 127.0)) * s["w_scale"])
    return (y if s["bias"] is None else y + s["bias"]).to(s["x"].dtype)


def _moments_plain(s):
    """sum over phases of scale x^T y, and of scale sum_c x, scale sum_c y, in float32."""
    (xd, xm), (yd, ym), (sd, sm) = ([t.float() for t in s["x"]], [t.float() for t in s["y"]], s["scale"])
    return ((xd.t() @ yd) * sd + (xm.t() @ ym) * sm, xd.sum(0) * sd + xm.sum(0) * sm,
            yd.sum(0) * sd + ym.sum(0) * sm)


def _philox(words, step):
    """Philox4x32-10 on counters (i, i >> 32, step, SALT), i < words: int64 [words, 4] of 32-bit values."""
    low = 0xFFFFFFFF
    i = torch.arange(words, device=DEVICE, dtype=torch.int64)
    x, y = i & low, i >> 32
    z, w = torch.full_like(i, step & low), torch.full_like(i, SALT)
    k0, k1 = SEED & low, SEED >> 32
    for _ in range(10):
        a, b = x * 0xD2511F53, z * 0xCD9E8D57
        x, y, z, w = ((b >> 32) & low) ^ y ^ k0, b & low, ((a >> 32) & low) ^ w ^ k1, a & low
        k0, k1 = (k0 + 0x9E3779B9) & low, (k1 + 0xBB67AE85) & low
    return torch.stack([x, y, z, w], 1)


def _encode(value, top, power, largest, u):
    """Codes q in 0..largest with value ~ q^power top / largest^power, rounded up with the probability that
    keeps the value's mean (u uniform); `top` is the block's largest value, 0 for a block held as zeros."""
    inv = torch.where(top > 0, torch.div(torch.full_like(top, float(largest**power)), top), 0.0)
    y = value * inv
    grid = (torch.arange(largest + 2, device=DEVICE, dtype=torch.float64) ** power).float()
    k = torch.bucketize(y, grid[: largest + 1], right=True) - 1
    up = u * (grid[k + 1] - grid[k]) < y - grid[k]
    return y, k, torch.where(up, k + 1, k).clamp(max=largest)


def _adamw_plain(s):
    """m = b1 m + (1 - b1) g; v = b2 v + (1 - b2) g^2; p = p (1 - lr wd) - lr / (1 - b1^t) m / (sqrt(v / (1 - b2^t)) + eps),
    over the flat buffers.  8-bit moments: m = +-q^2 max|m| / 127^2, v = q^4 max v / 255^4 per block of 256."""
    s["step"] += 1
    t = s["step"]
    narrow = s["case"]["bits"] == 8
    if narrow:
        c, d = s["m"].float().view(-1, BLOCK), s["v"].float().view(-1, BLOCK)
        m = ((c * c.abs()) * (s["m_scale"] * (1.0 / 127**2))[:, None]).view(-1)
        d2 = d * d
        v = ((d2 * d2) * (s["v_scale"] * (1.0 / 255**4))[:, None]).view(-1)
    else:
        m, v = s["m"], s["v"]
    g, p = s["grad"].float(), s["p"].float()
    m = m * BETA1 + g * (1.0 - BETA1)
    v = v * BETA2 + (g * g) * (1.0 - BETA2)
    denom = torch.sqrt(v) * (1.0 / math.sqrt(1.0 - BETA2**t)) + EPS
    s["p"].copy_(p * (1.0 - LR * DECAY) - torch.div(m, denom) * (LR / (1.0 - BETA1**t)))
    if not narrow:
        s["m"], s["v"] = m, v
        return {"p": s["p"], "exp_avg": m, "exp_avg_sq": v}
    r = _philox(m.numel() // 4, t).view(-1, BLOCK)
    um, uv = ((r & 0xFFFF).float() + 0.5) * 2.0**-16, ((r >> 16).float() + 0.5) * 2.0**-16
    m, v = m.view(-1, BLOCK), v.view(-1, BLOCK)
    top_v = v.amax(1, keepdim=True)
    top_v = torch.where(top_v >= 2.0**-90, top_v, 0.0)
    top_m = m.abs().amax(1, keepdim=True)
    top_m = torch.where((top_m >= 2.0**-100) & (top_v > 0), top_m, 0.0)
    _, _, qm = _encode(m.abs(), top_m, 2, 127, um)
    y, k, qv = _encode(v, top_v, 4, 255, uv)
    qv = torch.where(k == 0, (y > 0).to(qv.dtype), qv)
    qm = torch.where(m < 0, -qm, qm)
    s["m"], s["v"] = qm.to(torch.int8).view(-1), qv.to(torch.uint8).view(-1)
    s["m_scale"], s["v_scale"] = top_m.view(-1), top_v.view(-1)
    c, d2 = qm.float(), qv.float() * qv.float()
    return {"p": s["p"], "exp_avg": ((c * c.abs()) * (top_m * (1.0 / 127**2))).view(-1),
            "exp_avg_sq": ((d2 * d2) * (top_v * (1.0 / 255**4))).view(-1)}


def exact(case, seed):
    s = _inputs(case, seed)
    if case["op"] == "int8":
        # the whole numbers q are float32 decisions by definition; everything after them is in 64 bits
        top = s["x"].float().abs().max(1).values
        q = (s["x"].float() * (torch.full_like(top, 127.0) / top)[:, None]).round().double()
        unit = top.double() / 127
        y = torch.einsum("mk,nk->mn", q, s["w"].double()) * torch.outer(unit, s["w_scale"].double())
        return y if s["bias"] is None else y + s["bias"].double()[None, :]
    if case["op"] == "moments":
        w, bx, by = 0.0, 0.0, 0.0
        for x, y, scale in zip(s["x"], s["y"], (-1.0 / case["data"], 1.0 / case["model"])):
            x, y = x.double(), y.double()
            w = w + scale * torch.einsum("ci,cj->ij", x, y)
            bx, by = bx + scale * torch.einsum("ci->i", x), by + scale * torch.einsum("cj->j", y)
        return w, bx, by
    t, g, p = s["step"] + 1, s["grad"].double(), s["p"].double()
    if case["bits"] == 32:
        m, v = s["m"].double(), s["v"].double()
    else:
        unit_m = s["m_scale"].double().repeat_interleave(BLOCK) / 127**2
        unit_v = s["v_scale"].double().repeat_interleave(BLOCK) / 255**4
        m = s["m"].double().abs() * s["m"].double() * unit_m
        v = s["v"].double() ** 4 * unit_v
    m = m + (1 - BETA1) * (g - m)
    v = v + (1 - BETA2) * (g.square() - v)
    step = LR * (m / (1 - BETA1**t)) / ((v / (1 - BETA2**t)).sqrt() + EPS)
    p = p - LR * DECAY * p - step
    # an 8-bit moment is a rounding decided by a random word at float32 values: it has no 64-bit value
    narrow = case["bits"] == 8
    return {"p": p, "exp_avg": None if narrow else m, "exp_avg_sq": None if narrow else v}
