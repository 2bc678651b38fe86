"""Measured cases of the feed-forward, 8-bit and distillation operators of ``mpi_cuda_cnn_amd.ops``.

``listed()`` names the cases, ``draw()`` makes more of the same ranges, ``prepare()`` makes a case's inputs on the GPU,
``run()`` makes one pass over them: in elementary torch operations, or, with ``own`` set, through the framework's
operators.  ``exact()`` gives the same outputs from the definitions in 64 bits, ``work()`` what a pass has to move and
compute.

    gated   H = f(X Wg^T) * (X Wu^T)                              (forward; optionally with both projections saved)
    gated_bwd   dX, dWg, dWu from dH and the saved projections    (backward)
    i8      Y = f((Xq Wq^T) * sx * sw + b)                        (8-bit integer product, scales per token and channel)
    norm    S = X + R, 8-bit values and a scale per row of S / rms(S) * W
    distill temperature-softened divergence from a teacher's top logits, per row, and its gradient
"""

import math

import torch

own = False

_DT = {"bf16": torch.bfloat16, "fp32": torch.float32}


def _ops():
    import mpi_cuda_cnn_amd.ops as ops

    return ops


# ---------------------------------------------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------------------------------------------
def listed():
    return [
        # one token of a served block: the two weight matrices are read once, latency and bandwidth count
        {"name": "gated_token", "op": "gated", "m": 1, "d": 4096, "f": 8192, "act": "silu", "save": False},
        # a few sequences of odd total length through a small block
        {"name": "gated_ragged", "op": "gated", "m": 777, "d": 1024, "f": 2731, "act": "gelu", "save": True},
        # the forward pass of a training step: the projections are kept for the backward pass
        {"name": "gated_train", "op": "gated", "m": 8192, "d": 4096, "f": 12288, "act": "silu", "save": True},
        # the backward pass of a small block, rows and width odd
        {"name": "gated_bwd_ragged", "op": "gated_bwd", "m": 777, "d": 1024, "f": 2731, "act": "gelu"},
        # the backward pass of a training step
        {"name": "gated_bwd_train", "op": "gated_bwd", "m": 8192, "d": 4096, "f": 12288, "act": "silu"},
        # one token through a quantised projection
        {"name": "i8_token", "op": "i8", "m": 1, "n": 8192, "k": 4096, "act": "none", "bias": False, "out": "bf16"},
        # a batch of images at the 1000-class head behind a 4096-wide layer
        {"name": "i8_head", "op": "i8", "m": 640, "n": 1000, "k": 4096, "act": "none", "bias": True, "out": "fp32"},
        # a long prompt through a quantised projection
        {"name": "i8_prompt", "op": "i8", "m": 8192, "n": 12288, "k": 4096, "act": "relu", "bias": True, "out": "bf16"},
        # one token before its quantised projection
        {"name": "norm_token", "op": "norm", "m": 1, "d": 4096, "dtype": "bf16", "residual": True},
        # a long prompt before its quantised projection
        {"name": "norm_prompt", "op": "norm", "m": 16384, "d": 4096, "dtype": "bf16", "residual": True},
        # a batch of image classifiers' logits, 1000 classes
        {"name": "distill_classes", "op": "distill", "m": 640, "n": 1000, "k": 10, "t": 4.0, "dtype": "fp32"},
        # a training step over a large vocabulary
        {"name": "distill_vocab", "op": "distill", "m": 4096, "n": 120000, "k": 64, "t": 2.0, "dtype": "bf16"},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _width(rng, lo, hi):
    """A width between lo and hi: mostly of multiples of 64 or 8, one in four any number."""
    w = _log(rng, lo, hi)
    step = rng.choice([64, 64, 8, 1])
    return max(lo, w // step * step)


def draw(rng):
    op = rng.choice(["gated", "gated_bwd", "i8", "norm", "distill"])
    while True:
        if op in ("gated", "gated_bwd"):
            c = {"op": op, "m": _log(rng, 1, 8192), "d": _width(rng, 64, 8192), "f": _width(rng, 64, 16384),
                 "act": rng.choice(["silu", "silu", "gelu", "relu", "tanh", "none"])}
            if op == "gated":
                c["save"] = rng.random() < 0.5
            if c["m"] * c["d"] * c["f"] <= 8192 * 4096 * 12288:
                return c
        elif op == "i8":
            c = {"op": op, "m": _log(rng, 1, 8192), "n": _width(rng, 64, 16384), "k": _width(rng, 64, 16384),
                 "act": rng.choice(["none", "none", "relu", "tanh"]), "bias": rng.random() < 0.5,
                 "out": rng.choice(["bf16", "bf16", "fp32"])}
            if c["m"] * c["n"] * c["k"] <= 8192 * 12288 * 4096:
                return c
        elif op == "norm":
            c = {"op": op, "m": _log(rng, 1, 16384), "d": _width(rng, 64, 16384),
                 "dtype": rng.choice(["bf16", "bf16", "fp32"]), "residual": rng.random() < 0.75}
            if c["m"] * c["d"] <= 16384 * 4096:
                return c
        else:
            c = {"op": op, "m": _log(rng, 1, 4096), "n": _width(rng, 64, 250000), "k": _log(rng, 1, 64),
                 "t": rng.choice([1.0, 2.0, 4.0]), "dtype": rng.choice(["bf16", "bf16", "fp32"])}
            if c["m"] * c["n"] * (2 if c["dtype"] == "fp32" else 1) <= 4096 * 120000:
                return c


def work(case):
    op = case["op"]
    if op in ("gated", "gated_bwd"):
        m, d, f = case["m"], case["d"], case["f"]
        if op == "gated":
            return {"bytes": 2 * (m * d + 2 * f * d + m * f * (3 if case["save"] else 1)), "flops": 4 * m * d * f}
        return {"bytes": 2 * (3 * m * f + 2 * m * d + 4 * f * d), "flops": 8 * m * d * f}
    if op == "i8":
        m, n, k = case["m"], case["n"], case["k"]
        osz = 2 if case["out"] == "bf16" else 4
        return {"bytes": m * k + n * k + 4 * (m + n) + (4 * n if case["bias"] else 0) + osz * m * n, "flops": 2 * m * n * k}
    if op == "norm":
        m, d = case["m"], case["d"]
        es = 2 if case["dtype"] == "bf16" else 4
        n_in, n_out = (2, 1) if case["residual"] else (1, 0)
        return {"bytes": m * d * (es * (n_in + n_out) + 1) + es * d + 4 * m, "flops": 6 * m * d}
    m, n, k = case["m"], case["n"], case["k"]
    es = 2 if case["dtype"] == "bf16" else 4
    return {"bytes": 2 * es * m * n + (es + 8) * m * k + 4 * m, "flops": 6 * m * n}


# ---------------------------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------------------------
def _randn(g, *shape, std=1.0, dtype=torch.bfloat16):
    return (torch.randn(*shape, device="cuda", generator=g, dtype=torch.float32) * std).to(dtype)


def _randq(g, *shape):
    """8-bit values as a row's symmetric quantisation leaves them: a bell of about a quarter of the range."""
    return torch.randn(*shape, device="cuda", generator=g, dtype=torch.float32).mul_(32.0).round_().clamp_(-127, 127).to(torch.int8)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    s = dict(case)
    op = case["op"]
    if op in ("gated", "gated_bwd"):
        m, d, f = case["m"], case["d"], case["f"]
        s["x"] = _randn(g, m, d)
        # pre-activations of about unit size, as a trained block's are
        s["wg"] = _randn(g, f, d, std=d ** -0.5)
        s["wu"] = _randn(g, f, d, std=d ** -0.5)
        if op == "gated_bwd":
            # the two projections that the forward pass kept
            s["gate"] = (s["x"].float() @ s["wg"].float().t()).to(torch.bfloat16)
            s["up"] = (s["x"].float() @ s["wu"].float().t()).to(torch.bfloat16)
            s["dh"] = _randn(g, m, f, std=1e-2)
    elif op == "i8":
        m, n, k = case["m"], case["n"], case["k"]
        s["xq"], s["wq"] = _randq(g, m, k), _randq(g, n, k)
        s["sx"] = 0.01 + 0.04 * torch.rand(m, device="cuda", generator=g)
        s["sw"] = (0.01 + 0.02 * torch.rand(n, device="cuda", generator=g)) * k ** -0.5
        s["b"] = _randn(g, n, std=0.1, dtype=torch.float32) if case["bias"] else None
    elif op == "norm":
        m, d, dt = case["m"], case["d"], _DT[case["dtype"]]
        s["x"] = _randn(g, m, d, dtype=dt)
        # a residual stream has a few channels far larger than the others
        r = torch.randn(m, d, device="cuda", generator=g) * (1.0 + 20.0 * (torch.rand(d, device="cuda", generator=g) < 0.005))
        s["r"] = r.to(dt) if case["residual"] else None
        s["w"] = (1.0 + 0.1 * torch.randn(d, device="cuda", generator=g)).to(dt)
    else:
        m, n, k, dt = case["m"], case["n"], case["k"], _DT[case["dtype"]]
        s["z"] = _randn(g, m, n, std=2.0, dtype=dt)
        # the teacher's k largest: distinct classes, their logits falling, and the student leans to them as well
        step = max(1, n // k)
        at = torch.randint(0, step, (m, k), device="cuda", generator=g) + step * torch.arange(k, device="cuda")
        at = at[:, torch.randperm(k, device="cuda", generator=g)]
        top = torch.sort(torch.randn(m, k, device="cuda", generator=g) * 2.0 + 8.0, dim=1, descending=True).values
        s["z"].scatter_add_(1, at, (0.5 * top).to(dt))
        # shorter lists end in -1, and one row in sixteen has none (padding of the batch)
        have = torch.randint(max(1, k // 2), k + 1, (m, 1), device="cuda", generator=g)
        have[torch.rand(m, 1, device="cuda", generator=g) < 1 / 16] = 0
        s["ti"] = torch.where(torch.arange(k, device="cuda") < have, at, -1)
        s["tv"] = top.to(dt)
    return s


# ---------------------------------------------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------------------------------------------
def _act(v, act):
    if act == "silu":
        return v * torch.sigmoid(v)
    if act == "gelu":
        return 0.5 * v * (1.0 + torch.erf(v * math.sqrt(0.5)))
    if act == "relu":
        return torch.clamp(v, min=0.0)
    if act == "tanh":
        return torch.tanh(v)
    return v


def _act_and_slope(v, act):
    if act == "silu":
        s = torch.sigmoid(v)
        return v * s, s * (1.0 + v * (1.0 - s))
    if act == "gelu":
        c = 0.5 * (1.0 + torch.erf(v * math.sqrt(0.5)))
        return v * c, c + v * torch.exp(-0.5 * v * v) * (1.0 / math.sqrt(2.0 * math.pi))
    if act == "relu":
        on = (v > 0).to(v.dtype)
        return v * on, on
    if act == "tanh":
        t = torch.tanh(v)
        return t, 1.0 - t * t
    return v, torch.ones_like(v)


def _plain_gated(s):
    x = s["x"].float()
    g, u = x @ s["wg"].float().t(), x @ s["wu"].float().t()
    h = (_act(g, s["act"]) * u).to(torch.bfloat16)
    return {"h": h, "gate": g.to(torch.bfloat16), "up": u.to(torch.bfloat16)} if s["save"] else {"h": h}


def _plain_gated_bwd(s):
    dh, g, u = s["dh"].float(), s["gate"].float(), s["up"].float()
    a, da = _act_and_slope(g, s["act"])
    dg, du = dh * u * da, dh * a
    x = s["x"].float()
    dx = dg @ s["wg"].float() + du @ s["wu"].float()
    return {"dx": dx.to(torch.bfloat16), "dwg": (dg.t() @ x).to(torch.bfloat16), "dwu": (du.t() @ x).to(torch.bfloat16)}


def _plain_i8(s):
    y = (s["xq"].float() @ s["wq"].float().t()) * (s["sx"][:, None] * s["sw"][None, :])
    if s["b"] is not None:
        y = y + s["b"]
    return {"y": _act(y, s["act"]).to(_DT[s["out"]])}


def _values(q, scale):
    """What the 8-bit values stand for, each product rounded once to bf16."""
    return torch.mul(q, scale[:, None], out=torch.empty(q.shape, dtype=torch.bfloat16, device=q.device))


def _plain_norm(s):
    v = s["x"].float()
    if s["r"] is not None:
        v = v + s["r"].float()
    y = v * torch.rsqrt((v * v).mean(1, keepdim=True) + 1e-6) * s["w"].float()
    top = y.abs().amax(1, keepdim=True)
    q = torch.round(y * (127.0 / top)).clamp(-127, 127)
    scale = (top / 127.0)[:, 0]
    out = {"values": _values(q, scale), "scale": scale}
    if s["r"] is not None:
        out["sum"] = v.to(s["x"].dtype)
    return out


def _plain_distill(s):
    t = s["t"]
    z = s["z"].float() / t
    m = z.amax(1, keepdim=True)
    e = torch.exp(z - m)
    tot = e.sum(1, keepdim=True)
    lse = m + torch.log(tot)
    there = s["ti"] >= 0
    at = s["ti"].clamp(min=0)
    tv = (s["tv"].float() / t).masked_fill(~there, -math.inf)
    tm = tv.amax(1, keepdim=True)
    some = there.any(1, keepdim=True)
    tm = torch.where(some, tm, 0.0)
    te = torch.exp(tv - tm)
    ts = te.sum(1, keepdim=True)
    q = te / torch.where(some, ts, 1.0)
    logq = torch.where(there, tv - tm - torch.log(torch.where(some, ts, 1.0)), 0.0)
    logp = z.gather(1, at) - lse
    loss = (q * (logq - logp)).sum(1) * (t * t)
    d = (e / tot).scatter_add_(1, at, -q) * (_scale(s) * t)
    d = torch.where(some, d, 0.0)
    return {"dz": d.to(s["z"].dtype), "loss": loss}


def _scale(s):
    """The gradient is that of the rows' mean."""
    return 1.0 / s["m"]


def run(s):
    op = s["op"]
    if not own:
        return {"gated": _plain_gated, "gated_bwd": _plain_gated_bwd, "i8": _plain_i8, "norm": _plain_norm,
                "distill": _plain_distill}[op](s)
    ops = _ops()
    if op == "gated":
        if s["save"]:
            h, gate, up = ops.gated_linear(s["x"], s["wg"], s["wu"], s["act"], save=True)
            return {"h": h, "gate": gate, "up": up}
        return {"h": ops.gated_linear(s["x"], s["wg"], s["wu"], s["act"])}
    if op == "gated_bwd":
        dx, dwg, dwu = ops.gated_linear_bwd(s["dh"], s["x"], s["wg"], s["wu"], s["gate"], s["up"], s["act"])
        return {"dx": dx, "dwg": dwg, "dwu": dwu}
    if op == "i8":
        return {"y": ops.linear_i8(s["xq"], s["sx"], s["wq"], s["sw"], s["b"], s["act"], out_dtype=_DT[s["out"]])}
    if op == "norm":
        q, scale, v = ops.rmsnorm_i8(s["x"], s["w"], s["r"], eps=1e-6)
        out = {"values": _values(q, scale), "scale": scale}
        if s["r"] is not None:
            out["sum"] = v
        return out
    dz, loss = ops.distill_kl(s["z"], s["tv"], s["ti"], temperature=s["t"], scale=_scale(s))
    return {"dz": dz, "loss": loss}


# ---------------------------------------------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------------------------------------------
def _f64(v, act):
    """(f(v), f'(v)) in 64 bits."""
    if act == "silu":
        e = 1.0 / (1.0 + torch.exp(-v))
        return v * e, e + v * e * (1.0 - e)
    if act == "gelu":
        phi = torch.special.ndtr(v)
        return v * phi, phi + v * torch.exp(-v * v / 2.0) / math.sqrt(2.0 * math.pi)
    if act == "relu":
        return torch.where(v > 0, v, torch.zeros_like(v)), torch.where(v > 0, 1.0, 0.0).to(v.dtype)
    if act == "tanh":
        return torch.tanh(v), 1.0 / torch.cosh(v) ** 2
    return v, torch.ones_like(v)


def exact(case, seed):
    s = prepare(case, seed)
    op, D = case["op"], torch.float64
    if op == "gated":
        x = s["x"].to(D)
        g, u = torch.mm(x, s["wg"].to(D).t()), torch.mm(x, s["wu"].to(D).t())
        h = _f64(g, case["act"])[0] * u
        return {"h": h, "gate": g, "up": u} if case["save"] else {"h": h}
    if op == "gated_bwd":
        f, df = _f64(s["gate"].to(D), case["act"])
        dg = s["dh"].to(D) * s["up"].to(D) * df
        du = s["dh"].to(D) * f
        x = s["x"].to(D)
        return {"dx": torch.mm(dg, s["wg"].to(D)) + torch.mm(du, s["wu"].to(D)),
                "dwg": torch.mm(dg.t(), x), "dwu": torch.mm(du.t(), x)}
    if op == "i8":
        y = torch.mm(s["xq"].to(D), s["wq"].to(D).t()) * s["sx"].to(D)[:, None] * s["sw"].to(D)
        y = y if s["b"] is None else y + s["b"].to(D)
        return {"y": _f64(y, case["act"])[0]}
    if op == "norm":
        v = s["x"].to(D) if s["r"] is None else s["x"].to(D) + s["r"].to(D)
        y = v / torch.sqrt(v.square().mean(1, keepdim=True) + 1e-6) * s["w"].to(D)
        scale = y.abs().amax(1) / 127.0
        out = {"values": torch.round(y / scale[:, None]) * scale[:, None], "scale": scale}
        if s["r"] is not None:
            out["sum"] = v
        return out
    t, m, n = case["t"], case["m"], case["n"]
    dz = torch.empty(m, n, device="cuda", dtype=D)
    loss = torch.empty(m, device="cuda", dtype=D)
    step = max(1, (1 << 26) // n)
    for a in range(0, m, step):
        b = min(m, a + step)
        logp = torch.log_softmax(s["z"][a:b].to(D) / t, 1)
        ti = s["ti"][a:b]
        none = ti < 0
        tv = torch.where(none, torch.full_like(ti, -math.inf, dtype=D), s["tv"][a:b].to(D) / t)
        empty = none.all(1)
        tv[empty] = 0.0
        logq = torch.log_softmax(tv, 1)
        q = torch.where(none, 0.0, torch.exp(logq))
        term = torch.where(none, 0.0, q * (torch.where(none, 0.0, logq) - logp.gather(1, ti.clamp(min=0))))
        loss[a:b] = t * t * term.sum(1)
        d = torch.exp(logp)
        d.scatter_add_(1, ti.clamp(min=0), -q)
        d[empty] = 0.0
        dz[a:b] = d * (t / m)
    return {"dz": dz, "loss": loss}
