"""Cases that stand for what a user of this framework has its state-space, norm and gradient operators do, for timing.

Each case is one pass through a public entry point: ``selective_scan`` and ``causal_conv`` (sequences with and without
gradients, episode resets, single tokens with the state carried), ``rms_norm`` / ``rms_norm_fp8`` (the residual stream's
addition and norm) and ``clip_grad_norm_`` (a training step's gradients).  ``run`` computes them in plain torch operations, or
with ``own`` through the framework; ``exact`` steps through the definitions in 64 bits.  Sizes are those of the benchmark and
test configurations (learner unroll T=100 B=32, 48 actors, few-shot 128 x 128 tokens of 512, model dims 16 x 64, sequences
of 2048 and 8192), and odd ones in between.
"""
import math
import os
import sys

import torch

own = False


def _srwm():
    path = os.path.join(os.getcwd(), "modern-srwm_b200")
    if path not in sys.path:
        sys.path.insert(0, path)
    import srwm_b200
    return srwm_b200


def _scan(name, kind, B, L, D, S, dtype, G=1, done=False, gate=True):
    return {"name": name, "op": "scan", "kind": kind, "B": B, "L": L, "D": D, "S": S, "G": G, "done": done, "gate": gate,
            "dtype": dtype}


def _conv(name, kind, B, L, D, K, dtype, done=False):
    return {"name": name, "op": "conv", "kind": kind, "B": B, "L": L, "D": D, "K": K, "done": done, "dtype": dtype}


def _norm(name, kind, rows, D, dtype):
    return {"name": name, "op": "norm", "kind": kind, "rows": rows, "D": D, "dtype": dtype}


def _clip(name, tensors, total, dtype):
    return {"name": name, "op": "clip", "tensors": tensors, "total": total, "dtype": dtype}


def listed():
    return [
        # one environment step of 48 actors, hidden 256 widened twice, state advanced in place: latency
        _scan("scan actor step", "step", 48, 1, 512, 16, "f32"),
        # one token for many sequences served at once: the state's bytes
        _scan("scan token batch", "step", 256, 1, 2048, 16, "bf16"),
        # a lone long prompt: few channels, the time axis is the only thing to split
        _scan("scan long prompt", "prompt", 1, 8192, 1024, 16, "bf16"),
        # packed sequences (a reset at each start), two groups of B and C, wide states, odd sizes
        _scan("scan packed prompts", "prompt", 3, 1531, 1000, 64, "f32", G=2, done=True),
        # the learner's unroll with episode resets and a carried state, forward and backward
        _scan("scan unroll train", "train", 32, 100, 512, 16, "f32", done=True),
        # a training step's sequences: throughput
        _scan("scan train", "train", 8, 2048, 2048, 16, "bf16"),
        # the convolution in front of the scan: one actor step, the learner's unroll, the training step
        _conv("conv actor step", "step", 48, 1, 512, 4, "f32"),
        _conv("conv train", "train", 8, 2048, 2048, 4, "bf16"),
        # the few-shot model's rows (128 x 128 tokens of 512) with the residual's addition, forward and backward
        _norm("norm residual train", "train", 16384, 512, "f32"),
        # a served batch's rows, 8 bits out
        _norm("norm 8 bits", "fp8", 4099, 1024, "bf16"),
        # gradients of the agents' model, and of a large one
        _clip("clip agent", 24, 2500000, "f32"),
        _clip("clip large", 40, 160000000, "f32"),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.5)))))))


def draw(rng):
    """A case of the same kinds over the same ranges: lengths, batches and widths over their logarithm, odd ones among them."""
    most = {}
    for c in listed():
        most[c["op"]] = max(most.get(c["op"], 0), _cost(c))
    while True:
        op = rng.choice(("scan", "scan", "scan", "conv", "norm", "clip"))
        dtype = rng.choice(("f32", "bf16"))
        if op == "scan":
            kind = rng.choice(("step", "prompt", "train"))
            G = rng.choice((1, 1, 1, 2, 4))
            D = G * _log_int(rng, 24, 2100 // G)
            L = 1 if kind == "step" else _log_int(rng, 5, 8192)
            case = _scan("", kind, _log_int(rng, 1, 256 if kind == "step" else 32), L, D, rng.choice((8, 16, 16, 32, 64)), dtype, G,
                         kind != "step" and rng.random() < 0.4, rng.random() < 0.7)
        elif op == "conv":
            kind = rng.choice(("step", "prompt", "train"))
            L = 1 if kind == "step" else _log_int(rng, 5, 8192)
            case = _conv("", kind, _log_int(rng, 1, 256 if kind == "step" else 32), L, _log_int(rng, 24, 2100), rng.choice((2, 3, 4)),
                         dtype, kind != "step" and rng.random() < 0.4)
        elif op == "norm":
            case = _norm("", rng.choice(("train", "fp8", "plain")), _log_int(rng, 1, 16500), _log_int(rng, 24, 1100), dtype)
        else:
            case = _clip("", _log_int(rng, 1, 56), _log_int(rng, 20000, 160000000), dtype)
        del case["name"]
        if _cost(case) <= most[op]:
            return case


def _cost(case):
    w = work(case)
    return max(w["bytes"] / 6.5e12, w["flops"] / 7e13)


def work(case):
    """One pass: inputs read once, outputs written once; the recurrence's multiply-adds and exponentials."""
    s = 2 if case["dtype"] == "bf16" else 4
    if case["op"] == "scan":
        B, L, D, S, G = (case[k] for k in ("B", "L", "D", "S", "G"))
        rows, gate, train = B * L, 1 if case["gate"] else 0, case["kind"] == "train"
        flow = rows * (D * (3 + gate) + 2 * G * S) * s          # u, delta, z, B, C in, y out
        if train:                                               # dy in, their gradients out
            flow += rows * (D * (3 + gate) + 2 * G * S) * s
        state = 2 * B * D * S * 4 * (2 if train else 1)
        params = (D * S + 2 * D) * 4 * (2 if train else 1)
        return {"bytes": flow + state + params, "flops": rows * D * S * (24 if train else 7)}
    if case["op"] == "conv":
        B, L, D, K = (case[k] for k in ("B", "L", "D", "K"))
        train = case["kind"] == "train"
        return {"bytes": B * D * (L * (4 if train else 2) + (K - 1) * (4 if train else 2)) * s + D * (K + 1) * 4 * (2 if train else 1),
                "flops": B * L * D * (2 * K + 4) * (4 if train else 1)}
    if case["op"] == "norm":
        n, kind = case["rows"] * case["D"], case["kind"]
        out = {"plain": 2 * s, "train": 2 * s + 3 * s, "fp8": s + 1}[kind]
        return {"bytes": n * (2 * s + out) + case["D"] * 4 * (2 if kind == "train" else 1) + (case["rows"] * 4 if kind == "fp8" else 0),
                "flops": n * {"plain": 5, "train": 16, "fp8": 7}[kind]}
    return {"bytes": 2 * case["total"] * s, "flops": 3 * case["total"]}


# ---- inputs -----------------------------------------------------------------------------------------------------------------

class _Rand:
    """Seeded inputs made on the GPU."""

    def __init__(self, seed):
        self.g = torch.Generator(device="cuda")
        self.g.manual_seed(seed)

    def normal(self, *shape, dtype=torch.float32, scale=1.0):
        t = torch.empty(shape, device="cuda", dtype=torch.float32).normal_(generator=self.g)
        return (t.mul_(scale) if scale != 1.0 else t).to(dtype)

    def uniform(self, *shape):
        return torch.rand(shape, device="cuda", generator=self.g)


def _dt(case):
    return torch.bfloat16 if case["dtype"] == "bf16" else torch.float32


def _sizes(case):
    """A model's tensors: matrices of several sizes and vectors of odd lengths, `total` values in all."""
    n, total = case["tensors"], case["total"]
    share = [1.0 / (1 + (i * 7) % 5) if i % 3 else 0.002 for i in range(n)]
    sizes = [max(1, int(total * w / sum(share))) for w in share]
    return [v // 4 * 4 if i % 4 != 1 and v >= 64 else v for i, v in enumerate(sizes)]


def prepare(case, seed):
    r, dt, op = _Rand(seed), _dt(case), case["op"]
    train = case.get("kind") == "train"
    s = {"op": op, "kind": case.get("kind")}
    if op == "scan":
        B, L, D, S, G = (case[k] for k in ("B", "L", "D", "S", "G"))
        wide = r.normal(B, L, 2 * D, dtype=dt) if case["gate"] else None      # the input projection's rows: u's branch and the gate
        s["u"] = torch.nn.functional.silu(r.normal(B, L, D)).to(dt)
        s["z"] = wide[..., D:] if case["gate"] else None
        s["delta"] = r.normal(B, L, D, scale=0.5, dtype=dt)
        # step sizes between 0.001 and 0.1 at a raw value of zero, decays from 1 to S, as such layers are initialised
        step = torch.exp(math.log(1e-3) + r.uniform(D) * math.log(100.0))
        s["bias"] = step + torch.log(-torch.expm1(-step))
        s["A"] = -torch.arange(1, S + 1, device="cuda").float() * (1 + 0.1 * r.uniform(D, S))
        bc = r.normal(B, L, 2 * G * S, dtype=dt)
        s["B"], s["C"] = (t.reshape(B, L, G, S) if G > 1 else t for t in (bc[..., :G * S], bc[..., G * S:]))
        s["D"] = 1 + r.normal(D, scale=0.1)
        s["state"] = r.normal(B, D, S, scale=0.3)
        s["done"] = r.uniform(B, L) < max(0.02, 4.0 / L) if case["done"] else None
        if train:
            s["gout"], s["gstate"] = r.normal(B, L, D, dtype=dt), r.normal(B, D, S, scale=0.1)
            s["leaves"] = [k for k in ("u", "delta", "A", "B", "C", "D", "z", "bias", "state") if s[k] is not None]
            for k in s["leaves"]:
                s[k].requires_grad_()
    elif op == "conv":
        B, L, D, K = (case[k] for k in ("B", "L", "D", "K"))
        s["x"] = r.normal(B, L, 2 * D, dtype=dt)[..., :D]
        s["w"], s["bias"] = r.normal(D, K, scale=K ** -0.5), r.normal(D, scale=0.1)
        s["state"] = r.normal(B, K - 1, D, dtype=dt)
        s["done"] = r.uniform(B, L) < max(0.02, 4.0 / L) if case["done"] else None
        if train:
            s["gout"], s["gstate"] = r.normal(B, L, D, dtype=dt), r.normal(B, K - 1, D, dtype=dt)
            s["leaves"] = ["x", "w", "bias", "state"]
            for k in s["leaves"]:
                s[k].requires_grad_()
    elif op == "norm":
        rows, D = case["rows"], case["D"]
        s["x"], s["res"] = r.normal(rows, D, dtype=dt), r.normal(rows, D, scale=3.0, dtype=dt)
        s["w"] = 1 + r.normal(D, scale=0.1)
        if train:
            s["gout"], s["gres"] = r.normal(rows, D, dtype=dt), r.normal(rows, D, dtype=dt)
            s["leaves"] = ["x", "res", "w"]
            for k in s["leaves"]:
                s[k].requires_grad_()
    else:
        s["params"] = []
        for n in _sizes(case):
            p = torch.nn.Parameter(torch.empty(n, device="cuda", dtype=dt))
            p.grad = r.normal(n, dtype=dt, scale=0.02)
            s["params"].append(p)
        s["max_norm"] = 1.0
    return s


# ---- one pass ---------------------------------------------------------------------------------------------------------------

def run(s):
    if not own:
        return {"scan": _plain_scan, "conv": _plain_conv, "norm": _plain_norm, "clip": _plain_clip}[s["op"]](s)
    sb, kind = _srwm(), s["kind"]
    if s["op"] == "scan":
        args = (s["u"], s["delta"], s["A"], s["B"], s["C"])
        more = dict(D=s["D"], z=s["z"], delta_bias=s["bias"], state=s["state"], done=s["done"])
        if kind != "train":
            with torch.no_grad():
                return sb.selective_scan(*args, **more, inplace_state=kind == "step")
        y, state = sb.selective_scan(*args, **more)
        grads = torch.autograd.grad([y, state], [s[k] for k in s["leaves"]], [s["gout"], s["gstate"]])
        return y.detach(), state.detach(), list(grads)
    if s["op"] == "conv":
        more = dict(bias=s["bias"], state=s["state"], done=s["done"])
        if kind != "train":
            with torch.no_grad():
                return sb.causal_conv(s["x"], s["w"], **more, inplace_state=kind == "step")
        y, state = sb.causal_conv(s["x"], s["w"], **more)
        grads = torch.autograd.grad([y, state], [s[k] for k in s["leaves"]], [s["gout"], s["gstate"]])
        return y.detach(), state.detach(), list(grads)
    if s["op"] == "norm":
        if kind == "train":
            y, res = sb.rms_norm(s["x"], s["w"], residual=s["res"])
            grads = torch.autograd.grad([y, res], [s["x"], s["res"], s["w"]], [s["gout"], s["gres"]])
            return y.detach(), res.detach(), list(grads)
        with torch.no_grad():
            return (sb.rms_norm_fp8 if kind == "fp8" else sb.rms_norm)(s["x"], s["w"], residual=s["res"])
    norm = sb.clip_grad_norm_(s["params"], s["max_norm"])
    return norm, [p.grad for p in s["params"]]


# ---- plain forms ------------------------------------------------------------------------------------------------------------

def _steps(a, x):
    """h[t] = a[t] h[t-1] + x[t] along dimension 1, from zero: in doubling steps of the time axis."""
    a, h, k = a.clone(), x.clone(), 1
    while k < h.shape[1]:
        h[:, k:] = h[:, k:] + a[:, k:] * h[:, :-k]
        a[:, k:] = a[:, k:] * a[:, :-k]
        k *= 2
    return h


@torch.no_grad()
def _plain_scan(s):
    u, raw = s["u"].float(), s["delta"].float() + s["bias"]
    Bn, L, Dn = u.shape
    A, S = s["A"], s["A"].shape[1]

    def spread(t):      # [B, L, (G,) S] -> [B, L, D, S]
        t = t.float().reshape(Bn, L, -1, 1, S)
        return t.expand(-1, -1, -1, Dn // t.shape[2], -1).reshape(Bn, L, Dn, S)

    delta = torch.where(raw > 20, raw, torch.log1p(torch.exp(raw)))
    a = torch.exp(delta[..., None] * A)
    if s["done"] is not None:
        a = a * (~s["done"])[:, :, None, None]
    Bs, Cs = spread(s["B"]), spread(s["C"])
    x = (delta * u)[..., None] * Bs
    x[:, 0] += a[:, 0] * s["state"]
    h = _steps(a, x)
    del x
    pre = (h * Cs).sum(-1) + u * s["D"]
    y = pre
    if s["z"] is not None:
        z = s["z"].float()
        sig = torch.sigmoid(z)
        y = pre * z * sig
    y = y.to(s["u"].dtype)
    last = h[:, -1].contiguous()
    if s["kind"] == "step":
        s["state"].copy_(last)
        return y, s["state"]
    if s["kind"] != "train":
        return y, last
    go = s["gout"].float()
    dz = None
    if s["z"] is not None:
        dz = (go * pre * sig * (1 + z * (1 - sig))).to(s["z"].dtype)
        go = go * z * sig

    def gather(t):      # [B, L, D, S] -> the shape of B and C
        return t.reshape(Bn, L, -1, Dn // (s["B"].shape[2] if s["B"].dim() == 4 else 1), S).sum(3).reshape(s["B"].shape)

    dC = gather(go[..., None] * h).to(s["C"].dtype)
    g = go[..., None] * Cs
    g[:, -1] += s["gstate"]
    after = torch.cat([a[:, 1:], torch.zeros_like(a[:, :1])], 1)
    g = _steps(after.flip(1), g.flip(1)).flip(1)
    del after, Cs
    dstate = a[:, 0] * g[:, 0]
    before = torch.cat([s["state"][:, None], h[:, :-1]], 1)
    del h
    ga = g * a * before
    del before, a
    dA = (ga * delta[..., None]).sum((0, 1))
    gB = (g * Bs).sum(-1)
    dB = gather(g * (delta * u)[..., None]).to(s["B"].dtype)
    ddelta = u * gB + (ga * A).sum(-1)
    draw_ = ddelta * torch.sigmoid(raw)
    du = go * s["D"] + delta * gB
    grads = {"u": du.to(s["u"].dtype), "delta": draw_.to(s["delta"].dtype), "A": dA,
             "B": dB, "C": dC, "D": (go * u).sum((0, 1)), "z": dz, "bias": draw_.sum((0, 1)), "state": dstate}
    return y, last, [grads[k] for k in s["leaves"]]


def _taps(s, L, K):
    """For each tap: where in [state, x] it reads, and whether no reset lies between there and the output's step."""
    if s["done"] is None:
        return [(K - 1 - i, None) for i in range(K)], None
    seg = torch.cumsum(s["done"], 1)
    ext = torch.cat([torch.zeros_like(seg[:, :1]).expand(-1, K - 1), seg], 1)
    return [(K - 1 - i, (ext[:, K - 1 - i:K - 1 - i + L] == seg)[..., None]) for i in range(K)], (ext[:, L:] == seg[:, -1:])[..., None]


@torch.no_grad()
def _plain_conv(s):
    w, dt = s["w"], s["x"].dtype
    L, K = s["x"].shape[1], w.shape[1]
    rows = torch.cat([s["state"], s["x"]], 1)
    ext = rows.float()
    taps, keep = _taps(s, L, K)
    parts = [ext[:, at:at + L] if ok is None else ext[:, at:at + L] * ok for at, ok in taps]
    pre = s["bias"] + sum(p * w[:, at] for p, (at, _) in zip(parts, taps))
    sig = torch.sigmoid(pre)
    y = (pre * sig).to(dt)
    last = rows[:, L:] if keep is None else rows[:, L:] * keep
    if s["kind"] == "step":
        s["state"].copy_(last.clone())
        return y, s["state"]
    if s["kind"] != "train":
        return y, last.contiguous()
    g = s["gout"].float() * sig * (1 + pre * (1 - sig))
    dw = torch.stack([(g * p).sum((0, 1)) for p in parts][::-1], 1)
    dext = torch.zeros_like(ext)
    for at, ok in taps:
        dext[:, at:at + L] += (g if ok is None else g * ok) * w[:, at]
    dext[:, L:] += s["gstate"].float() if keep is None else s["gstate"].float() * keep
    return y, last.contiguous(), [dext[:, K - 1:].to(dt), dw, g.sum((0, 1)), dext[:, :K - 1].to(dt)]


@torch.no_grad()
def _plain_norm(s):
    w, dt = s["w"], s["x"].dtype
    res = (s["x"].float() + s["res"].float()).to(dt)
    f = res.float()
    rstd = torch.rsqrt((f * f).mean(-1, keepdim=True) + 1e-6)
    xh = f * rstd
    y = xh * w
    if s["kind"] == "fp8":
        scale = torch.clamp(y.abs().amax(-1, keepdim=True) / 448.0, min=2.0 ** -126)
        return (y / scale).to(torch.float8_e4m3fn), scale, res
    if s["kind"] != "train":
        return y.to(dt), res
    gy = s["gout"].float()
    g = gy * w
    d = (rstd * (g - xh * (g * xh).mean(-1, keepdim=True)) + s["gres"].float()).to(dt)
    return y.to(dt), res, [d, d.clone(), (gy * xh).sum(0)]


@torch.no_grad()
def _plain_clip(s):
    grads = [p.grad for p in s["params"]]
    norm = torch.sqrt(sum((g.float() * g.float()).sum() for g in grads))
    coef = torch.clamp(s["max_norm"] / (norm + 1e-6), max=1.0)
    for g in grads:
        g.copy_(g.float() * coef)
    return norm, grads


# ---- the definitions, step by step in 64 bits -------------------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        return {"scan": _exact_scan, "conv": _exact_conv, "norm": _exact_norm, "clip": _exact_clip}[case["op"]](case, s)


def _exact_scan(case, s):
    B, L, D, S, G = (case[k] for k in ("B", "L", "D", "S", "G"))
    if B * L * D * S * 8 > 24e9:
        return None
    d = {k: v.detach().double() for k, v in s.items() if isinstance(v, torch.Tensor) and k != "done"}
    group = torch.arange(D, device="cuda") // (D // G)
    Bm, Cm = (d[k].reshape(B, L, G, S) for k in ("B", "C"))
    raw = d["delta"] + d["bias"]
    delta = torch.nn.functional.softplus(raw, threshold=40)
    live = torch.ones(B, L, device="cuda", dtype=torch.float64) if s["done"] is None else (~s["done"]).double()
    train, A = case["kind"] == "train", d["A"]
    h, pre = d["state"], torch.empty(B, L, D, device="cuda", dtype=torch.float64)
    hist = torch.empty(L + 1, B, D, S, device="cuda", dtype=torch.float64) if train else None
    if train:
        hist[0] = h
    for t in range(L):
        a = torch.exp(delta[:, t, :, None] * A) * live[:, t, None, None]
        h = a * h + (delta[:, t] * d["u"][:, t])[..., None] * Bm[:, t][:, group]
        pre[:, t] = torch.einsum("bds,bds->bd", h, Cm[:, t][:, group]) + d["D"] * d["u"][:, t]
        if train:
            hist[t + 1] = h
    gate = d["z"] / (1 + torch.exp(-d["z"])) if case["gate"] else torch.ones_like(pre)
    y = pre * gate
    if not train:
        return y, h
    go = d["gout"] * gate
    out = {k: torch.zeros_like(d[k]) for k in s["leaves"]}
    if case["gate"]:
        sig = 1 / (1 + torch.exp(-d["z"]))
        out["z"] = d["gout"] * pre * (sig + d["z"] * sig * (1 - sig))
    g = d["gstate"].clone()
    dBm, dCm = torch.zeros_like(Bm), torch.zeros_like(Cm)
    for t in reversed(range(L)):
        dl, ut = delta[:, t, :, None], d["u"][:, t, :, None]
        Bt, Ct = Bm[:, t][:, group], Cm[:, t][:, group]
        g = g + go[:, t, :, None] * Ct
        dCm[:, t].index_add_(1, group, go[:, t, :, None] * hist[t + 1])
        dBm[:, t].index_add_(1, group, g * dl * ut)
        a = torch.exp(dl * A) * live[:, t, None, None]
        ga = g * a * hist[t]
        out["A"] += (ga * dl).sum(0)
        gB = (g * Bt).sum(-1)
        out["u"][:, t] = go[:, t] * d["D"] + delta[:, t] * gB
        out["delta"][:, t] = ((ga * A).sum(-1) + gB * d["u"][:, t]) / (1 + torch.exp(-raw[:, t]))
        g = a * g
    out["state"], out["B"], out["C"] = g, dBm.reshape(d["B"].shape), dCm.reshape(d["C"].shape)
    out["D"], out["bias"] = (go * d["u"]).sum((0, 1)), out["delta"].sum((0, 1))
    return y, h, [out[k] for k in s["leaves"]]


def _exact_conv(case, s):
    B, L, D, K = (case[k] for k in ("B", "L", "D", "K"))
    if B * L * D * 8 * K > 24e9:
        return None
    leaves = [s[k].detach().double().requires_grad_() for k in ("x", "w", "bias", "state")]
    with torch.enable_grad():
        x, w, bias, state = leaves
        window, outs = state, []
        if s["done"] is None:                       # the same for every sequence: all windows at once
            rows = torch.cat([state, x], 1)
            pre, last = torch.einsum("bldk,dk->bld", rows.unfold(1, K, 1), w) + bias, rows[:, L:]
        else:
            live = (~s["done"]).double()[..., None, None]
            for t in range(L):                      # a step at a time, the window emptied at each reset
                window = torch.cat([window * live[:, t], x[:, t:t + 1]], 1)
                outs.append(torch.einsum("bkd,dk->bd", window, w) + bias)
                window = window[:, 1:]
            pre, last = torch.stack(outs, 1), window
        y = pre / (1 + torch.exp(-pre))
        if case["kind"] != "train":
            return y.detach(), last.detach()
        grads = torch.autograd.grad([y, last], leaves, [s["gout"].double(), s["gstate"].double()])
    return y.detach(), last.detach(), list(grads)


def _exact_norm(case, s):
    res = (s["x"].double() + s["res"].double()).to(_dt(case))          # the stream as it is stored
    leaf, w = res.detach().double().requires_grad_(), s["w"].detach().double().requires_grad_()
    with torch.enable_grad():
        y = leaf / torch.sqrt((leaf ** 2).mean(-1, keepdim=True) + 1e-6) * w
        if case["kind"] == "train":
            dres, dw = torch.autograd.grad(y, [leaf, w], s["gout"].double())
            d = dres + s["gres"].double()
            return y.detach(), res.double(), [d, d, dw]
    y = y.detach()
    if case["kind"] == "plain":
        return y, res.double()
    scale = y.abs().amax(-1, keepdim=True) / 448
    return (y / scale).clamp(-448, 448).to(torch.float8_e4m3fn).double(), scale, res.double()


def _exact_clip(case, s):
    grads = [p.grad.double() for p in s["params"]]
    norm = sum(float((g ** 2).sum()) for g in grads) ** 0.5
    return torch.tensor(norm, dtype=torch.float64), [g * min(1.0, s["max_norm"] / (norm + 1e-6)) for g in grads]
