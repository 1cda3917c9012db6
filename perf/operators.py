"""The dense feed-forward operators (`dense.py`) as benchmark cases: residual addition + root-mean-square norm, matrix product with bias,
activation and residual, gated projection.

`listed()` and `draw()` give cases, `prepare()` the inputs of one, `run()` makes one pass: with `own` the calls a user makes of the package,
without it the same operator from elementary torch operations in 32 bits.  `exact()` is the operator in 64 bits."""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
EPS = 1e-6


# ------------------------------------------------------------------ cases
def listed():
    return [
        # one token of a decode step: the residual joins, the normed row leaves in 8 bits for the block-scaled products
        {"name": "norm quant decode", "op": "norm_quant", "rows": 1, "dim": 4096, "dtype": "bf16", "wdtype": "bf16", "residual": True},
        # a prefill chunk with a ragged number of tokens at the larger hidden size of the model family
        {"name": "norm quant prefill", "op": "norm_quant", "rows": 4099, "dim": 5120, "dtype": "bf16", "wdtype": "fp32", "residual": True},
        # a training step's norm over packed sequences: forward and backward, the norm weight kept in 32 bits
        {"name": "norm train", "op": "norm_train", "rows": 8191, "dim": 4096, "dtype": "bf16", "wdtype": "fp32", "residual": True},
        # the down projection of one decoded token with the residual added
        {"name": "linear decode", "op": "linear", "m": 1, "n": 4096, "k": 2048, "dtype": "bf16", "act": "none", "bias": False, "residual": True},
        # a head of odd width on a feature size that no vector load divides
        {"name": "linear odd", "op": "linear", "m": 333, "n": 1001, "k": 2310, "dtype": "fp16", "act": "gelu", "bias": True, "residual": True},
        # a wide projection over a prefill chunk
        {"name": "linear prefill", "op": "linear", "m": 4096, "n": 12288, "k": 4096, "dtype": "bf16", "act": "gelu", "bias": True, "residual": False},
        # FP8 weights and activations: a small decode batch
        {"name": "linear q8 decode", "op": "linear_q8", "m": 8, "n": 4096, "k": 4096, "act": "silu", "bias": True, "residual": True},
        # FP8 weights and activations: the down projection of a prefill chunk with the residual added
        {"name": "linear q8 prefill", "op": "linear_q8", "m": 4096, "n": 4096, "k": 2048, "act": "none", "bias": False, "residual": True},
        # a training step of one projection: forward, and the gradients of input, weight, bias and residual
        {"name": "linear train", "op": "linear_train", "m": 2039, "n": 4096, "k": 4096, "dtype": "fp16", "act": "gelu_tanh", "bias": True, "residual": True},
        # gate and up projections of a decode batch of four tokens
        {"name": "gated decode", "op": "gated", "m": 4, "inter": 2048, "k": 4096, "dtype": "bf16", "act": "silu", "limit": 10.0},
        # the same over a prefill chunk
        {"name": "gated prefill", "op": "gated", "m": 4096, "inter": 2048, "k": 4096, "dtype": "bf16", "act": "silu", "limit": 10.0},
        # a training step of the gated projection: forward, and the gradients of input and weights
        {"name": "gated train", "op": "gated_train", "m": 4001, "inter": 2304, "k": 5120, "dtype": "bf16", "act": "silu", "limit": 0.0},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["norm_quant", "norm_train", "linear", "linear", "linear_q8", "linear_train", "gated", "gated", "gated_train"])
    dtype = rng.choice(["bf16", "bf16", "fp16"])
    if kind in ("norm_quant", "norm_train"):
        step = 32 if kind == "norm_quant" else rng.choice([1, 8, 8])
        dim = max(step, _log(rng, 64, 8192) // step * step)
        return {"op": kind, "rows": _log(rng, 1, 6000), "dim": dim, "dtype": dtype, "wdtype": rng.choice([dtype, "fp32"]), "residual": rng.random() < 0.8}
    m = _log(rng, 1, 3000) if not kind.endswith("train") else _log(rng, 64, 2500)
    act = rng.choice(["none", "relu", "silu", "gelu", "gelu_tanh"])
    if kind == "linear_q8":
        return {"op": kind, "m": m, "n": 16 * _log(rng, 16, 512), "k": 128 * _log(rng, 2, 40), "act": act, "bias": rng.random() < 0.5, "residual": rng.random() < 0.7}
    step = 1 if rng.random() < 0.15 else 8  # now and then a width that no vector load divides
    k = max(step, _log(rng, 256, 6000) // step * step)
    if kind.startswith("gated"):
        inter = max(step, _log(rng, 128, 3000) // step * step)
        return {"op": kind, "m": m, "inter": inter, "k": k, "dtype": dtype, "act": rng.choice(["silu", "silu", "gelu", "gelu_tanh", "relu"]), "limit": rng.choice([0.0, 10.0])}
    n = max(step, _log(rng, 256, 8192) // step * step)
    return {"op": kind, "m": m, "n": n, "k": k, "dtype": dtype, "act": act, "bias": rng.random() < 0.5, "residual": rng.random() < 0.6}


def work(c):
    op = c["op"]
    if op.startswith("norm"):
        e = 4 if c["dtype"] == "fp32" else 2
        n = c["rows"] * c["dim"]
        wb = c["dim"] * (4 if c["wdtype"] == "fp32" else 2)
        res = 2 if c["residual"] else 0  # the residual is read and the sum is written
        if op == "norm_quant":
            return {"bytes": n * e * (1 + res) + n + n // 32 + wb, "flops": 6 * n}
        # forward: x, residual in, y, sum out; backward: the two gradients in, one gradient out for both (x and residual are still at hand)
        return {"bytes": n * e * (2 + res) + n * e * (2 + (1 if c["residual"] else 0)) + 2 * wb, "flops": 16 * n}
    if op.startswith("gated"):
        m, i, k = c["m"], c["inter"], c["k"]
        b, f = 2 * (m * k + 2 * i * k + m * i), 4 * m * i * k
        return {"bytes": b, "flops": f} if op == "gated" else {"bytes": b + 2 * (m * i + m * k + 2 * i * k), "flops": 3 * f}
    m, n, k = c["m"], c["n"], c["k"]
    extra = (2 * m * n if c["residual"] else 0) + (2 * n if c["bias"] else 0)
    if op == "linear_q8":
        return {"bytes": m * k + m * (k // 32) + n * k + (-(-n // 32)) * (k // 32) + 2 * m * n + extra, "flops": 2 * m * n * k}
    b, f = 2 * (m * k + n * k + m * n) + extra, 2 * m * n * k
    return {"bytes": b, "flops": f} if op == "linear" else {"bytes": b + 2 * (m * n + m * k + n * k) + (2 * n if c["bias"] else 0), "flops": 3 * f}


# ------------------------------------------------------------------ inputs
def _e4m3_blocks(v, rows):
    """fp32 [N, K] -> (e4m3 bytes [N, K], E8M0 bytes [ceil(N / rows), K / 32]): one power-of-two scale per rows x 32 block."""
    n, k = v.shape
    nb = -(-n // rows)
    full = torch.zeros(nb * rows, k, device=v.device)
    full[:n] = v
    b = full.view(nb, rows, k // 32, 32)
    e = torch.ceil(torch.log2(b.abs().amax(dim=(1, 3)).clamp_min(1e-4) / 448.0) - 1e-6)
    q = (b / torch.exp2(e)[:, None, :, None]).clamp(-448, 448).view(nb * rows, k)[:n]
    return q.to(torch.float8_e4m3fn).view(torch.uint8).contiguous(), (e + 127).to(torch.uint8).contiguous()


def prepare(c, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(int(seed))
    rnd = lambda *s: torch.randn(*s, generator=g, device=dev)  # noqa: E731
    st, op = dict(c), c["op"]
    if op.startswith("norm"):
        dt, r, d = DTYPES[c["dtype"]], c["rows"], c["dim"]
        channel = torch.exp(0.5 * rnd(d))  # hidden states: some channels are several times larger than the rest
        st["x"] = (rnd(r, d) * channel).to(dt)
        st["residual_in"] = (2.0 * rnd(r, d) * channel).to(dt) if c["residual"] else None
        st["weight"] = (1.0 + 0.2 * rnd(d)).to(DTYPES[c["wdtype"]])
        if op == "norm_train":
            st["gy"] = (0.1 * rnd(r, d)).to(dt)
            st["gs"] = (0.1 * rnd(r, d)).to(dt) if c["residual"] else None
            for n in ("x", "residual_in", "weight"):
                if st[n] is not None:
                    st[n].requires_grad_(True)
        return st
    m, k = c["m"], c["k"]
    if op == "linear_q8":
        st["x8"], st["xsf"] = _e4m3_blocks(rnd(m, k), 1)
        st["w8"], st["s8"] = _e4m3_blocks(rnd(c["n"], k) / math.sqrt(k), 32)
        dt = torch.bfloat16
    else:
        dt = DTYPES[c["dtype"]]
        st["x"] = rnd(m, k).to(dt)
        rows = 2 * c["inter"] if op.startswith("gated") else c["n"]
        st["w"] = (rnd(rows, k) * (2.0 if op.startswith("gated") else 1.0) / math.sqrt(k)).to(dt)
    width = c["inter"] if op.startswith("gated") else c["n"]
    if not op.startswith("gated"):
        st["b"] = (0.5 * rnd(width)).to(dt) if c["bias"] else None
        st["res"] = rnd(m, width).to(dt) if c["residual"] else None
    if op.endswith("train"):
        st["gy"] = (0.1 * rnd(m, width)).to(dt)
        for n in ("x", "w", "b", "res"):
            if st.get(n) is not None:
                st[n].requires_grad_(True)
    return st


# ------------------------------------------------------------------ one pass
def _dense():
    from __graft_entry__ import load_package
    load_package()
    import dsv41_b200.dense as dense
    return dense


def run(st):
    if own:
        return _run_own(st)
    with torch.no_grad():
        return _run_plain(st)


def _run_own(st):
    D, op = _dense(), st["op"]
    act = None if st.get("act") == "none" else st.get("act")
    if op == "norm_quant":
        q8, sf, s = D.add_rms_norm_quant(st["x"], st["residual_in"], st["weight"], EPS)
        return {"q": q8.view(torch.float8_e4m3fn), "scale": sf.view(torch.float8_e8m0fnu), "sum": s if st["residual"] else None}
    if op == "norm_train":
        y, s = D.add_rms_norm(st["x"], st["residual_in"], st["weight"], EPS)
        if st["residual"]:
            dx, dr, dw = torch.autograd.grad((y, s), (st["x"], st["residual_in"], st["weight"]), (st["gy"], st["gs"]))
            return {"y": y, "sum": s, "dx": dx, "dresidual": dr, "dweight": dw}
        dx, dw = torch.autograd.grad(y, (st["x"], st["weight"]), st["gy"])
        return {"y": y, "dx": dx, "dweight": dw}
    if op == "linear_q8":
        return {"y": D.linear_act_q8(st["x8"], st["xsf"], st["w8"], st["s8"], bias=st["b"], act=act, residual=st["res"])}
    if op == "gated":
        return {"h": D.gated_linear(st["x"], st["w"], act=act, limit=st["limit"])}
    if op == "linear":
        return {"y": D.linear_act(st["x"], st["w"], bias=st["b"], act=act, residual=st["res"])}
    if op == "gated_train":
        h = D.gated_linear(st["x"], st["w"], act=act, limit=st["limit"])
        dx, dw = torch.autograd.grad(h, (st["x"], st["w"]), st["gy"])
        return {"h": h, "dx": dx, "dw": dw}
    y = D.linear_act(st["x"], st["w"], bias=st["b"], act=act, residual=st["res"])
    names = [n for n in ("x", "w", "b", "res") if st[n] is not None]
    return {"y": y, **{"d" + n: t for n, t in zip(names, torch.autograd.grad(y, [st[n] for n in names], st["gy"]))}}


def _act(name, z):
    """act(z) and act'(z)."""
    if name == "relu":
        return z.clamp_min(0), (z > 0).to(z.dtype)
    if name == "silu":
        s = 1 / (1 + torch.exp(-z))
        return z * s, s * (1 + z * (1 - s))
    if name == "gelu":
        p = 0.5 * (1 + torch.erf(z * math.sqrt(0.5)))
        return z * p, p + z * torch.exp(-0.5 * z * z) / math.sqrt(2 * math.pi)
    if name == "gelu_tanh":
        a = math.sqrt(2 / math.pi)
        t = torch.tanh(a * (z + 0.044715 * z * z * z))
        return 0.5 * z * (1 + t), 0.5 * (1 + t) + 0.5 * z * (1 - t * t) * a * (1 + 3 * 0.044715 * z * z)
    return z, torch.ones_like(z)


def _quantise(y):
    """fp32 [R, D] -> e4m3 values and the power-of-two scale of each 32: the smallest one that brings the group's largest value to 448 or less."""
    b = y.view(y.shape[0], -1, 32)
    amax = b.abs().amax(-1).clamp_min(1e-4)
    mant, e = torch.frexp(amax)  # amax = mant * 2^e, 448 = 0.875 * 2^9
    scale = torch.exp2((e - 9 + (mant > 0.875).to(e.dtype)).float())
    return (b / scale.unsqueeze(-1)).to(torch.float8_e4m3fn).view(y.shape), scale.to(torch.float8_e8m0fnu)


def _value8(codes, scale_bytes, rows):
    """Bytes of e4m3 with one E8M0 scale per rows x 32 block as fp32."""
    n = codes.shape[0]
    s = torch.exp2(scale_bytes.float() - 127.0).repeat_interleave(32, dim=1)
    return codes.view(torch.float8_e4m3fn).float() * s.repeat_interleave(rows, dim=0)[:n]


def _run_plain(st):
    op = st["op"]
    if op.startswith("norm"):
        dt = st["x"].dtype
        s = st["x"].float()
        if st["residual"]:
            s = s + st["residual_in"].float()
        w = st["weight"].float()
        rinv = torch.rsqrt((s * s).mean(-1, keepdim=True) + EPS)
        n = s * rinv
        y = n * w
        if op == "norm_quant":
            q, scale = _quantise(y)
            return {"q": q, "scale": scale, "sum": s.to(dt) if st["residual"] else None}
        gy = st["gy"].float()
        gw = gy * w
        dx = rinv * (gw - n * (gw * n).mean(-1, keepdim=True))
        dw = (gy * n).sum(0).to(st["weight"].dtype)
        if not st["residual"]:
            return {"y": y.to(dt), "dx": dx.to(dt), "dweight": dw}
        dx = (dx + st["gs"].float()).to(dt)
        return {"y": y.to(dt), "sum": s.to(dt), "dx": dx, "dresidual": dx, "dweight": dw}
    if op.startswith("gated"):
        dt, x, w, i = st["x"].dtype, st["x"].float(), st["w"].float(), st["inter"]
        gu = x @ w.t()
        g, u = gu[:, :i], gu[:, i:]
        lim = st["limit"]
        gc, uc = (g.clamp(max=lim), u.clamp(-lim, lim)) if lim > 0 else (g, u)
        a, da = _act(st["act"], gc)
        h = (a * uc).to(dt)
        if op == "gated":
            return {"h": h}
        gy = st["gy"].float()
        dg, du = gy * uc * da, gy * a
        if lim > 0:
            dg, du = dg * (g <= lim), du * (u.abs() <= lim)
        dgu = torch.cat([dg, du], dim=1)
        return {"h": h, "dx": (dgu @ w).to(dt), "dw": (dgu.t() @ x).to(dt)}
    if op == "linear_q8":
        dt, x, w = torch.bfloat16, _value8(st["x8"], st["xsf"], 1), _value8(st["w8"], st["s8"], 32)
    else:
        dt, x, w = st["x"].dtype, st["x"].float(), st["w"].float()
    z = x @ w.t()
    if st["bias"]:
        z = z + st["b"].float()
    y, da = _act(st["act"], z)
    if st["residual"]:
        y = y + st["res"].float()
    out = {"y": y.to(dt)}
    if op == "linear_train":
        dz = st["gy"].float() * da
        out["dx"], out["dw"] = (dz @ w).to(dt), (dz.t() @ x).to(dt)
        if st["bias"]:
            out["db"] = dz.sum(0).to(dt)
        if st["residual"]:
            out["dres"] = st["gy"]
    return out


# ------------------------------------------------------------------ the operators in 64 bits
def _act64(name, z):
    if name == "relu":
        return torch.where(z > 0, z, torch.zeros_like(z))
    if name == "silu":
        return z * torch.sigmoid(z)
    if name == "gelu":
        return z * torch.special.ndtr(z)
    if name == "gelu_tanh":
        return z * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3))  # (1 + tanh a) / 2 = sigmoid(2 a)
    return z


def exact(c, seed):
    st = prepare(c, seed)
    op = c["op"]

    def leaf(n):
        t = st.get(n)
        return None if t is None else t.detach().double().requires_grad_(op.endswith("train"))

    def grads(outs, leaves, gs):
        names = [n for n in leaves if leaves[n] is not None]
        return dict(zip(names, torch.autograd.grad(outs, [leaves[n] for n in names], gs)))

    if op.startswith("norm"):
        x, r, w = leaf("x"), leaf("residual_in"), leaf("weight")
        s = x if r is None else x + r
        y = w * s / torch.sqrt(s.square().sum(-1, keepdim=True) / c["dim"] + EPS)
        if op == "norm_quant":
            groups = y.reshape(c["rows"], c["dim"] // 32, 32)
            top = groups.abs().max(-1).values.clamp_min(float(torch.tensor(1e-4))) / 448
            e = torch.floor(torch.log2(top)) - 1
            for _ in range(3):  # the smallest power of two that is not below top, without trusting the logarithm's last bit
                e = torch.where(torch.exp2(e) < top, e + 1, e)
            v = groups / torch.exp2(e)[..., None]
            step = torch.exp2(torch.floor(torch.log2(v.abs().clamp_min(2.0 ** -6))) - 3)  # the grid of e4m3 around v
            q = torch.clamp(torch.round(v / step) * step, -448, 448)
            return {"q": q.reshape(y.shape), "scale": torch.exp2(e), "sum": s if r is not None else None}
        d = grads((y, s) if r is not None else (y,), {"dx": x, "dresidual": r, "dweight": w},
                  (st["gy"].double(), st["gs"].double()) if r is not None else (st["gy"].double(),))
        return {"y": y.detach(), **({"sum": s.detach()} if r is not None else {}), **d}
    if op == "linear_q8":
        up = lambda q, s, rows: q.view(torch.float8_e4m3fn).double() * torch.pow(2.0, s.double() - 127).repeat_interleave(rows, 0)[: q.shape[0]].repeat_interleave(32, 1)  # noqa: E731
        x, w = up(st["x8"], st["xsf"], 1), up(st["w8"], st["s8"], 32)
    else:
        x, w = leaf("x"), leaf("w")
    z = torch.nn.functional.linear(x, w)
    if op.startswith("gated"):
        g, u = z.split(c["inter"], dim=1)
        if c["limit"] > 0:
            g, u = torch.clamp(g, max=c["limit"]), torch.clamp(u, -c["limit"], c["limit"])
        h = _act64(c["act"], g) * u
        return {"h": h.detach(), **(grads(h, {"dx": x, "dw": w}, st["gy"].double()) if op == "gated_train" else {})}
    b, r = leaf("b"), leaf("res")
    if b is not None:
        z = z + b
    y = _act64(c["act"], z)
    if r is not None:
        y = y + r
    return {"y": y.detach(), **(grads(y, {"dx": x, "dw": w, "db": b, "dres": r}, st["gy"].double()) if op == "linear_train" else {})}
