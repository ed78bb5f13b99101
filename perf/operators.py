"""The cases by which the gated recurrence and the group norm with an activation are measured.

Five kinds of pass:

* ``step``        one token per sequence through the gated recurrence (decode);
* ``scan``        the recurrence over whole sequences, forward only (prefill);
* ``scan_train``  the same with its gradient;
* ``norm``        group norm + activation, channels last, forward only;
* ``norm_train``  the same with its gradient.

``own`` selects the framework's operators; otherwise each pass is computed in its plain form, by
elementary torch operations in 32 bits.  ``exact`` evaluates the definitions in 64 bits.
"""
import math

import torch

own = False

_TYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
_EPS = 1e-5


# ------------------------------------------------------------------------------- cases
def listed():
    return [
        # decode of one sequence at the 12-layer model's width: nothing but latency
        dict(name="step_one", kind="step", dtype="bf16", B=1, D=768),
        # decode of a full serving batch at a wide state
        dict(name="step_batch", kind="step", dtype="bf16", B=256, D=2048),
        # prefill of one long prompt at the 12-layer model's length and width
        dict(name="scan_prefill", kind="scan", dtype="bf16", B=1, L=32768, D=768, reset=False, h0=False),
        # the same length at the Block's d_state: very few channels, all the parallelism is in time
        dict(name="scan_narrow", kind="scan", dtype="bf16", B=1, L=32768, D=64, reset=False, h0=True),
        # a short prompt, odd length
        dict(name="scan_short", kind="scan", dtype="bf16", B=2, L=257, D=256, reset=False, h0=True),
        # a training step at the 24-layer model's batch and length, the state somewhat wider than the model
        dict(name="scan_train", kind="scan_train", dtype="bf16", B=8, L=4096, D=1280, reset=False, h0=False),
        # fp32 training on packed documents of ragged lengths, odd sizes, state carried between windows
        dict(name="scan_train_packed", kind="scan_train", dtype="f32", B=3, L=1537, D=333, reset=True, h0=True),
        # the layer's norm of each head and token over a long prompt
        dict(name="norm_heads", kind="norm", dtype="bf16", N=32768, S=1, C=768, G=12, act="silu"),
        # the same in a training step at the 24-layer model's sizes
        dict(name="norm_heads_train", kind="norm_train", dtype="bf16", N=32768, S=1, C=1024, G=16, act="silu"),
        # a feature map of 64 x 64 positions, groups of 10 channels
        dict(name="norm_map", kind="norm", dtype="bf16", N=16, S=4096, C=320, G=32, act="silu"),
        # a training step on larger maps in fp32
        dict(name="norm_map_train", kind="norm_train", dtype="f32", N=4, S=16384, C=128, G=32, act="silu"),
        # a small map without an activation, odd position count
        dict(name="norm_small_train", kind="norm_train", dtype="bf16", N=2, S=225, C=96, G=8, act="none"),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["step", "scan", "scan", "scan_train", "scan_train", "norm", "norm", "norm_train", "norm_train"])
    dtype = rng.choice(["bf16", "bf16", "f32"])
    room = (48 << 20) // (2 if dtype == "bf16" else 4)  # elements of one activation
    if kind == "step":
        return dict(kind=kind, dtype=dtype, B=_log_int(rng, 1, 256), D=_log_int(rng, 16, 4096))
    if kind.startswith("scan"):
        D = _log_int(rng, 16, 4096)
        if rng.random() < 0.6:
            D = max(16, D // 16 * 16)
        B = _log_int(rng, 1, 16)
        L = _log_int(rng, 1, min(65536, room // (B * D)))
        return dict(kind=kind, dtype=dtype, B=B, L=L, D=D, reset=rng.random() < 0.4, h0=rng.random() < 0.5)
    G = rng.choice([1, 2, 3, 4, 8, 12, 16, 32])
    C = G * max(1, min(2048 // G, _log_int(rng, 2, 256)))
    if rng.random() < 0.4:
        S, N = 1, _log_int(rng, 1, min(65536, room // C))
    else:
        S = _log_int(rng, 2, min(65536, room // C))
        N = _log_int(rng, 1, max(1, min(64, room // (C * S))))
    return dict(kind=kind, dtype=dtype, N=N, S=S, C=C, G=G, act=rng.choice(["silu", "silu", "none"]))


# ------------------------------------------------------------------------------- inputs
def prepare(case, seed):
    dev = "cuda"
    g = torch.Generator(device=dev).manual_seed(seed)
    dt = _TYPES[case["dtype"]]

    def normal(*shape):
        return torch.randn(*shape, generator=g, device=dev)

    s = {"case": case}
    kind = case["kind"]
    if kind in ("step", "scan", "scan_train"):
        B, D = case["B"], case["D"]
        rows = (B,) if kind == "step" else (B, case["L"])
        # the decay gate as the layer initialises it: softplus(bias) log-spread over 0.001 .. 0.1,
        # moved by what the projection adds
        d0 = 0.001 + 0.099 * torch.rand(D, generator=g, device=dev)
        projs = normal(*rows, 3 * D)
        projs[..., :D] = torch.log(torch.expm1(d0)) + 0.5 * projs[..., :D]
        s["projs"] = projs.to(dt)
        s["A_log"] = torch.log(torch.linspace(0.99, 0.9999, D, device=dev))
        s["h0"] = normal(B, D) if kind == "step" or case["h0"] else None
        s["D"] = D
        if kind == "step":
            s["h_next"] = torch.empty(B, D, device=dev)
            return s
        # packed documents of some 200 tokens each
        s["reset"] = torch.rand(B, case["L"], generator=g, device=dev) < 0.005 if case["reset"] else None
        if kind == "scan_train":
            s["dy"] = normal(B, case["L"], D).to(dt)
            s["dh"] = normal(B, D) if case["h0"] else None  # the next window's gradient
            s["projs"].requires_grad_()
            s["A_log"].requires_grad_()
            if case["h0"]:
                s["h0"].requires_grad_()
        return s
    N, S, C = case["N"], case["S"], case["C"]
    s["x"] = (normal(N, S, C) * (0.5 + torch.rand(C, generator=g, device=dev)) + 0.3 * normal(C)).to(dt)
    s["w"] = (1.0 + 0.1 * normal(C)).to(dt)
    s["b"] = (0.1 * normal(C)).to(dt)
    if kind == "norm_train":
        s["dy"] = normal(N, S, C).to(dt)
        for k in ("x", "w", "b"):
            s[k].requires_grad_()
    return s


# ------------------------------------------------------------------------------- one pass
def run(state):
    if own:
        return _run_own(state)
    with torch.no_grad():
        kind = state["case"]["kind"]
        if kind == "step":
            return _plain_step(state)
        if kind == "scan":
            return _plain_scan(state)
        if kind == "scan_train":
            return _plain_scan_train(state)
        return _plain_norm(state, kind == "norm_train")


def _run_own(s):
    from hdcmamba_b200 import ops, recurrent

    case = s["case"]
    kind = case["kind"]
    if kind == "step":
        y, h = ops.gated_step(s["projs"], s["A_log"], s["h0"], s["D"], h_out=s["h_next"])
        return {"y": y, "h": h}
    if kind == "scan":
        y, h = ops.gated_scan(s["projs"], s["A_log"], s["D"], h0=s["h0"], reset=s["reset"])
        return {"y": y, "h": h}
    if kind == "scan_train":
        y, h = recurrent.gated_scan(s["projs"], s["A_log"], s["D"], h0=s["h0"], reset=s["reset"])
        wrt = [s["projs"], s["A_log"]] + ([s["h0"]] if case["h0"] else [])
        outs, douts = ([y, h], [s["dy"], s["dh"]]) if case["h0"] else ([y], [s["dy"]])
        grads = torch.autograd.grad(outs, wrt, douts)
        return {"y": y, "h": h, "dprojs": grads[0], "dA_log": grads[1], "dh0": grads[2] if case["h0"] else None}
    if kind == "norm":
        return {"y": ops.group_norm_act(s["x"], case["G"], s["w"], s["b"], eps=_EPS, act=case["act"])}
    y = recurrent.group_norm_act(s["x"], case["G"], s["w"], s["b"], eps=_EPS, act=case["act"])
    dx, dw, db = torch.autograd.grad([y], [s["x"], s["w"], s["b"]], [s["dy"]])
    return {"y": y, "dx": dx, "dw": dw, "db": db}


# plain forms: 32 bits throughout, rounded once at the end
def _terms(projs, A_log, D):
    """d = softplus(dt), A = -exp(A_log), a = exp(d A), and the raw dt, x, b in 32 bits."""
    p = projs.float()
    dt, x, b = p[..., :D], p[..., D:2 * D], p[..., 2 * D:]
    d = dt.clamp(min=0) + torch.log1p(torch.exp(-dt.abs()))
    A = -torch.exp(A_log)
    return dt, x, b, d, A, torch.exp(d * A)


def _plain_step(s):
    _, x, b, d, _, a = _terms(s["projs"], s["A_log"], s["D"])
    h = a * s["h0"] + d * b * x
    return {"y": h.to(s["projs"].dtype), "h": h}


def _recur(a, u):
    """h_t = a_t h_{t-1} + u_t along dim 1, from zero: spans of 1, 2, 4, ... steps joined pairwise."""
    k = 1
    while k < u.shape[1]:
        u = torch.cat([u[:, :k], u[:, k:] + a[:, k:] * u[:, :-k]], 1)
        a = torch.cat([a[:, :k], a[:, k:] * a[:, :-k]], 1)
        k *= 2
    return u


def _plain_forward(s):
    dt, x, b, d, A, a = _terms(s["projs"], s["A_log"], s["D"])
    if s["reset"] is not None:
        a = a * (~s["reset"]).unsqueeze(-1)
    u = d * b * x
    if s["h0"] is not None:
        u[:, 0] += a[:, 0] * s["h0"]
    return dt, x, b, d, A, a, _recur(a, u)


def _plain_scan(s):
    h = _plain_forward(s)[-1]
    return {"y": h.to(s["projs"].dtype), "h": h[:, -1]}


def _plain_scan_train(s):
    dt, x, b, d, A, a, h = _plain_forward(s)
    typ = s["projs"].dtype
    h0 = s["h0"] if s["h0"] is not None else torch.zeros_like(h[:, 0])
    g = s["dy"].float()
    if s["dh"] is not None:
        g = torch.cat([g[:, :-1], g[:, -1:] + s["dh"].unsqueeze(1)], 1)
    a_next = torch.cat([a[:, 1:], torch.zeros_like(a[:, :1])], 1)
    g = _recur(a_next.flip(1), g.flip(1)).flip(1)
    before = torch.cat([h0.unsqueeze(1), h[:, :-1]], 1)
    along = g * a * before  # the gradient of log a
    dd = along * A + g * b * x
    dprojs = torch.cat([dd * torch.sigmoid(dt), g * d * b, g * d * x], -1)
    return {"y": h.to(typ), "h": h[:, -1], "dprojs": dprojs.to(typ), "dA_log": (along * d * A).sum((0, 1)),
            "dh0": a[:, 0] * g[:, 0] if s["h0"] is not None else None}


def _plain_norm(s, train):
    case, typ = s["case"], s["x"].dtype
    N, S, C, G = case["N"], case["S"], case["C"], case["G"]
    x = s["x"].float().reshape(N, S, G, C // G)
    w, b = s["w"].float(), s["b"].float()
    mean = x.mean((1, 3), keepdim=True)
    centred = x - mean
    rstd = torch.rsqrt(centred.square().mean((1, 3), keepdim=True) + _EPS)
    xh = (centred * rstd).reshape(N, S, C)
    z = xh * w + b
    silu = case["act"] == "silu"
    sig = torch.sigmoid(z) if silu else None
    out = {"y": (z * sig if silu else z).to(typ)}
    if train:
        dz = s["dy"].float()
        if silu:
            dz = dz * sig * (1.0 + z * (1.0 - sig))
        e = (dz * w).reshape(N, S, G, C // G)
        xg = xh.reshape(N, S, G, C // G)
        dx = rstd * (e - e.mean((1, 3), keepdim=True) - xg * (e * xg).mean((1, 3), keepdim=True))
        out |= {"dx": dx.reshape(N, S, C).to(typ), "dw": (dz * xh).sum((0, 1)).to(typ), "db": dz.sum((0, 1)).to(typ)}
    return out


# ------------------------------------------------------------------------------- the definitions in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        return _exact_recurrence(s) if "D" in case else _exact_norm(s)


def _exact_recurrence(s):
    """One token after another, as the recurrence is written."""
    case, D = s["case"], s["D"]
    step = case["kind"] == "step"
    p = s["projs"].double()
    dt, x, b = (p.unsqueeze(1) if step else p).split(D, -1)
    L = dt.shape[1]
    rate = s["A_log"].double().exp()
    gate = torch.logaddexp(dt, torch.zeros_like(dt))
    keep = torch.exp(-gate * rate)
    if not step and s["reset"] is not None:
        keep.masked_fill_(s["reset"].unsqueeze(-1), 0.0)
    start = s["h0"].double() if s["h0"] is not None else torch.zeros_like(dt[:, 0])
    fed = gate * x * b
    y = torch.empty_like(dt)
    h = start
    for t in range(L):
        h = torch.addcmul(fed[:, t], keep[:, t], h)
        y[:, t] = h
    if step:
        return {"y": y[:, 0], "h": h}
    if case["kind"] == "scan":
        return {"y": y, "h": h}
    g = s["dy"].double()
    carry = s["dh"].double() if s["dh"] is not None else torch.zeros_like(start)
    for t in range(L - 1, -1, -1):
        g[:, t] += carry
        carry = keep[:, t] * g[:, t]
    # the state that each step kept: keep_t h_{t-1}
    kept = y - fed
    kept[:, 0] = keep[:, 0] * start
    kept[:, 1:] = keep[:, 1:] * y[:, :-1]
    by_log_keep = g * kept
    by_gate = g * x * b - by_log_keep * rate
    dprojs = torch.cat([by_gate / (1.0 + torch.exp(-dt)), g * gate * b, g * gate * x], -1)
    return {"y": y, "h": h, "dprojs": dprojs, "dA_log": -(by_log_keep * gate).sum((0, 1)) * rate,
            "dh0": carry if s["h0"] is not None else None}


def _exact_norm(s):
    """Group by group, the definition and its derivative by the chain rule."""
    case = s["case"]
    N, S, C, G = case["N"], case["S"], case["C"], case["G"]
    per = C // G
    x = s["x"].double()
    w, b = s["w"].double(), s["b"].double()
    train = case["kind"] == "norm_train"
    names = ("y", "dx", "dw", "db") if train else ("y",)
    out = {k: torch.empty(x.shape if k in ("y", "dx") else w.shape, dtype=torch.float64, device=x.device) for k in names}
    for k in range(G):
        cut = slice(k * per, (k + 1) * per)
        xs = x[..., cut].reshape(N, S * per)
        var, mean = torch.var_mean(xs, 1, correction=0, keepdim=True)
        sd = torch.sqrt(var + _EPS)
        n = ((xs - mean) / sd).reshape(N, S, per)
        z = torch.addcmul(b[cut], n, w[cut])
        y = z / (1.0 + torch.exp(-z)) if case["act"] == "silu" else z
        out["y"][..., cut] = y
        if not train:
            continue
        dz = s["dy"][..., cut].double()
        if case["act"] == "silu":
            q = 1.0 / (1.0 + torch.exp(-z))
            dz = dz * (q + y * (1.0 - q))
        out["dw"][cut] = torch.einsum("nsc,nsc->c", dz, n)
        out["db"][cut] = dz.sum((0, 1))
        dn = (dz * w[cut]).reshape(N, -1)
        flat = n.reshape(N, -1)
        dx = dn - dn.mean(1, keepdim=True) - flat * (dn * flat).mean(1, keepdim=True)
        out["dx"][..., cut] = (dx / sd).reshape(N, S, per)
    return out


# ------------------------------------------------------------------------------- work
def work(case):
    es = 2 if case["dtype"] == "bf16" else 4
    kind = case["kind"]
    if kind == "step":
        n, D = case["B"] * case["D"], case["D"]
        return {"bytes": n * (4 * es + 8) + 4 * D, "flops": 12 * n}
    if kind.startswith("scan"):
        B, L, D = case["B"], case["L"], case["D"]
        n = B * L * D
        small = 4 * D + 4 * B * D * (2 if case["h0"] else 1) + (B * L if case["reset"] else 0)
        if kind == "scan":
            return {"bytes": 4 * n * es + small, "flops": 12 * n}
        # projs and dy read once, y and dprojs written once
        return {"bytes": 8 * n * es + 2 * small, "flops": 40 * n}
    n, C = case["N"] * case["S"] * case["C"], case["C"]
    if kind == "norm":
        return {"bytes": 2 * n * es + 2 * C * es, "flops": 14 * n}
    # x and dy read once, y and dx written once
    return {"bytes": 4 * n * es + 4 * C * es, "flops": 40 * n}
