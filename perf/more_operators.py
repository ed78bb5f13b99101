"""The cases by which decayed linear attention, the token embedding and gradient clipping are measured.

Six kinds of pass:

* ``attn_step``    one token per sequence through the attention's state (decode);
* ``attn``         whole sequences, forward only (prefill), with the state after them;
* ``attn_train``   the same with its gradients;
* ``embed``        lookup of a prompt's rows, scaled;
* ``embed_train``  the lookup with the gradient of its table;
* ``clip``         the norm over all gradients of a model, and the gradients scaled to it.

``own`` selects the framework's operators; otherwise each pass is computed in its plain form, by
elementary torch operations in 32 bits (sums of squares in 64).  ``exact`` evaluates the
definitions in 64 bits.
"""
import math

import torch

own = False

_TYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
_CHUNK = 128  # tokens that the plain attention takes at a time


# ------------------------------------------------------------------------------- cases
def listed():
    return [
        # decode of one sequence at the 12-layer model's heads: latency
        dict(name="step_one", kind="attn_step", dtype="bf16", B=1, H=12, D=64),
        # decode of a full serving batch at the 24-layer model's heads: the states' traffic
        dict(name="step_batch", kind="attn_step", dtype="bf16", B=256, H=16, D=64),
        # prefill of one long prompt at the 12-layer model's length and heads
        dict(name="prefill_long", kind="attn", dtype="bf16", B=1, L=32768, H=12, D=64, state=False),
        # a short prompt of odd length that goes on from a state, at the small model's heads
        dict(name="prefill_short", kind="attn", dtype="bf16", B=2, L=257, H=8, D=32, state=True),
        # a training step at the 24-layer model's batch, length and heads
        dict(name="attn_train", kind="attn_train", dtype="bf16", B=8, L=4096, H=16, D=64, state=False),
        # fp32 training window by window, odd length, wide heads of a size that is no power of two
        dict(name="attn_train_window", kind="attn_train", dtype="f32", B=3, L=1537, H=4, D=96, state=True),
        # the lookup of the long prompt
        dict(name="embed_prompt", kind="embed", dtype="bf16", N=32768, V=50304, D=768, ids="zipf", scaled=False),
        # a training step of the 24-layer model's embedding on text: few ids take most of the tokens
        dict(name="embed_train", kind="embed_train", dtype="bf16", N=32768, V=50304, D=1024, ids="zipf", scaled=True),
        # the small model's in fp32, a batch of which a third is padding, all of it one id
        dict(name="embed_train_small", kind="embed_train", dtype="f32", N=512, V=4096, D=256, ids="padded", scaled=False),
        # all gradients of the 12-layer model in bf16, clipped
        dict(name="clip_model", kind="clip", dtype="bf16", layers=12, dm=768, ds=64, heads=12, V=50304, norm=3.0),
        # the 24-layer model with matrices in bf16 and vectors in fp32, small enough to stay as they are
        dict(name="clip_mixed", kind="clip", dtype="mixed", layers=24, dm=1024, ds=128, heads=16, V=50304, norm=0.5),
        # the small model in fp32: many tensors, little data
        dict(name="clip_small", kind="clip", dtype="f32", layers=2, dm=256, ds=64, heads=8, V=4096, norm=3.0),
    ]


def _log_int(rng, lo, hi):
    hi = max(lo, hi)
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["attn_step", "attn", "attn", "attn_train", "attn_train", "embed", "embed_train", "embed_train", "clip"])
    dtype = rng.choice(["bf16", "bf16", "f32"])
    if kind == "clip":
        heads = rng.choice([2, 4, 8, 12, 16])
        return dict(kind=kind, dtype=rng.choice(["bf16", "f32", "mixed"]), layers=_log_int(rng, 1, 16),
                    dm=heads * _log_int(rng, 4, 48), ds=_log_int(rng, 16, 128), heads=heads, V=_log_int(rng, 256, 50304),
                    norm=rng.choice([0.5, 3.0, 30.0]))
    if kind.startswith("embed"):
        D = _log_int(rng, 16, 2048)
        if rng.random() < 0.6:
            D = max(16, D // 16 * 16)
        wide = 1 if dtype == "bf16" else 2
        return dict(kind=kind, dtype=dtype, N=_log_int(rng, 1, min(65536, (32 << 20) // (D * wide))),
                    V=_log_int(rng, 64, min(131072, (48 << 20) // (D * wide))), D=D,
                    ids=rng.choice(["zipf", "uniform", "padded"]), scaled=rng.random() < 0.5)
    H = rng.choice([1, 2, 3, 4, 8, 12, 16, 24])
    D = rng.choice([16, 32, 32, 40, 64, 64, 64, 80, 96, 128, rng.randint(8, 128)])
    if kind == "attn_step":
        return dict(kind=kind, dtype=dtype, B=_log_int(rng, 1, max(1, (16 << 20) // (H * D * D))), H=H, D=D)
    # the work of a head grows with its size: fewer elements for wide heads, and for 32-bit ones
    room = (24 << 20) * 64 // max(64, D) // (1 if dtype == "bf16" else 4)
    B = _log_int(rng, 1, 16)
    return dict(kind=kind, dtype=dtype, B=B, L=_log_int(rng, 1, min(32768, room // (B * H * D))), H=H, D=D,
                state=rng.random() < 0.5)


# ------------------------------------------------------------------------------- inputs
def _shapes(case):
    """The shapes of a language model's parameters, matrices and vectors apart (Block by Block)."""
    dm, ds, V = case["dm"], case["ds"], case["V"]
    P = 3 * ds + 4 * dm
    matrices = [(V, dm)] + [(dm, 1, 4), (P, dm), (dm, ds + dm)] * case["layers"]
    vectors = [(dm,), (dm,), (dm,), (P,), (ds,), (case["heads"],), (dm,), (dm,)] * case["layers"] + [(dm,)] * 4
    return matrices, vectors


def _token_ids(case, g, dev):
    N, V = case["N"], case["V"]
    u = torch.rand(N, generator=g, device=dev, dtype=torch.float64)
    if case["ids"] == "zipf":  # the k-th most frequent id has a share of 1 / (k + 2.7)
        share = 1.0 / (torch.arange(V, device=dev, dtype=torch.float64) + 2.7)
        top = torch.cumsum(share, 0)
        ids = torch.searchsorted(top, u * top[-1])
    else:
        ids = (u * V).long()
    if case["ids"] == "padded":
        ids = torch.where(torch.rand(N, generator=g, device=dev) < 0.33, 0, ids)
    return ids.clamp_(max=V - 1)


def _views(flat, shapes):
    at, out = 0, []
    for s in shapes:
        n = math.prod(s)
        out.append(flat[at:at + n].view(s))
        at += n
    return out


def prepare(case, seed):
    dev = "cuda"
    g = torch.Generator(device=dev).manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, generator=g, device=dev)

    s = {"case": case}
    kind = case["kind"]
    if kind == "clip":
        matrices, vectors = _shapes(case)
        # gradients lie one behind the other in one buffer per type; so do the clipped ones
        parts = [("bf16", matrices), ("f32", vectors)] if case["dtype"] == "mixed" else [(case["dtype"], matrices + vectors)]
        total = sum(math.prod(x) for x in matrices + vectors)
        s["grads"], s["outs"], s["flat_outs"] = [], [], []
        for name, shapes in parts:
            n = sum(math.prod(x) for x in shapes)
            flat = (normal(n) * (case["norm"] / math.sqrt(total))).to(_TYPES[name])
            clipped = torch.empty_like(flat)
            s["grads"] += _views(flat, shapes)
            s["outs"] += _views(clipped, shapes)
            s["flat_outs"].append(clipped)
        s["max_norm"] = 1.0
        return s
    dt = _TYPES[case["dtype"]]
    D = case["D"]
    if kind.startswith("embed"):
        s["ids"] = _token_ids(case, g, dev)
        s["weight"] = (0.02 * normal(case["V"], D)).to(dt)
        s["scale"] = math.sqrt(D) if case["scaled"] else 1.0
        if kind == "embed_train":
            s["dy"] = normal(case["N"], D).to(dt)
            s["weight"].requires_grad_()
        return s
    B, H = case["B"], case["H"]
    rows = (B, H, D) if kind == "attn_step" else (B, case["L"], H, D)
    for k in ("q", "k", "v"):
        s[k] = normal(*rows).to(dt)
    # decays of 0.6 to 0.9995 a token: heads that remember two tokens to two thousand
    low, high = math.log(0.0005), math.log(0.5)
    s["log_decay"] = -torch.exp(low + (high - low) * torch.rand(H, generator=g, device=dev))
    s["scale"] = D ** -0.5
    if kind == "attn_step":
        s["state"] = normal(B, H, D, D)
        s["state_next"] = torch.empty_like(s["state"])
        return s
    s["state"] = normal(B, H, D, D) if case["state"] else None
    if kind == "attn_train":
        s["do"] = normal(*rows).to(dt)
        s["dstate"] = normal(B, H, D, D) if case["state"] else None  # the next window's gradient
        for k in ("q", "k", "v"):
            s[k].requires_grad_()
        if case["state"]:
            s["state"].requires_grad_()
    return s


# ------------------------------------------------------------------------------- one pass
def run(state):
    if own:
        return _run_own(state)
    with torch.no_grad():
        kind = state["case"]["kind"]
        if kind == "clip":
            return _plain_clip(state)
        if kind.startswith("embed"):
            return _plain_embed(state)
        if kind == "attn_step":
            return _plain_step(state)
        return _plain_attn(state)


def _run_own(s):
    from hdcmamba_b200 import ops, recurrent, training

    case = s["case"]
    kind = case["kind"]
    if kind == "attn_step":
        o, state = ops.decay_attention_step(s["q"], s["k"], s["v"], s["log_decay"], s["state"], scale=s["scale"],
                                            state_out=s["state_next"])
        return {"o": o, "state": state}
    if kind == "attn":
        o, state = ops.decay_attention(s["q"], s["k"], s["v"], s["log_decay"], scale=s["scale"], state=s["state"])
        return {"o": o, "state": state}
    if kind == "attn_train":
        o, state = recurrent.decay_attention(s["q"], s["k"], s["v"], s["log_decay"], scale=s["scale"], state=s["state"])
        wrt = [s["q"], s["k"], s["v"]] + ([s["state"]] if case["state"] else [])
        outs, douts = ([o, state], [s["do"], s["dstate"]]) if case["state"] else ([o], [s["do"]])
        grads = torch.autograd.grad(outs, wrt, douts)
        return {"o": o, "state": state, "dq": grads[0], "dk": grads[1], "dv": grads[2],
                "dstate": grads[3] if case["state"] else None}
    if kind == "embed":
        return {"y": ops.embedding(s["ids"], s["weight"], scale=s["scale"])}
    if kind == "embed_train":
        y = training.embedding(s["ids"], s["weight"], scale=s["scale"])
        (dw,) = torch.autograd.grad([y], [s["weight"]], [s["dy"]])
        return {"y": y, "dweight": dw}
    norm = ops.clip_grads(s["grads"], s["max_norm"], out=s["outs"])
    return {"norm": norm, "clipped": s["flat_outs"]}


# plain forms: 32 bits throughout, rounded once at the end
def _plain_step(s):
    q, k, v = s["q"].float(), s["k"].float(), s["v"].float()
    keep = torch.exp(s["log_decay"])[:, None, None]
    state = keep * s["state"] + k.unsqueeze(-1) * v.unsqueeze(-2)
    o = s["scale"] * (q.unsqueeze(-1) * state).sum(-2)
    return {"o": o.to(s["q"].dtype), "state": state}


def _spans(states, keep):
    """S_n = keep S_{n-1} + states_n along dim 2, from zero: spans of 1, 2, 4, ... joined pairwise."""
    k = 1
    while k < states.shape[2]:
        states = torch.cat([states[:, :, :k], states[:, :, k:] + keep * states[:, :, :-k]], 2)
        keep = keep * keep
        k *= 2
    return states


def _attend(q, k, v, g, first, last):
    """o_t = q_t S_t with S_t = exp(g) S_{t-1} + k_t v_t, chunk by chunk; all [B, H, L, D] in 32 bits.
    first: the state before the sequence or None.  Returns (o, the state after it or None)."""
    B, H, L, D = q.shape
    C = min(_CHUNK, L)
    N = -(-L // C)
    q, k, v = (torch.nn.functional.pad(x, (0, 0, 0, N * C - L)).view(B, H, N, C, D) for x in (q, k, v))
    t = torch.arange(C, device=q.device)
    g = g[:, None, None]
    apart = t[:, None] - t
    mask = torch.where(apart >= 0, torch.exp(g * apart.clamp(min=0)), 0.0)[:, None]
    o = ((q @ k.transpose(-1, -2)) * mask) @ v
    add = (k * torch.exp(g * (C - 1 - t))[..., None]).transpose(-1, -2) @ v
    keep = torch.exp(g * C)[..., None]
    if first is not None:
        add = torch.cat([first.unsqueeze(2), add], 2)
    after = _spans(add, keep)
    before = after[:, :, :N] if first is not None else torch.cat([torch.zeros_like(after[:, :, :1]), after[:, :, :-1]], 2)
    o = o + (q @ before) * torch.exp(g * (t + 1))[..., None]
    state = None
    if last:  # rows behind the sequence add nothing, but the state must not decay over them
        own_rows = L - (N - 1) * C
        w = torch.exp(g * (own_rows - 1 - t).clamp(min=0))[..., 0, :, None]
        state = torch.exp(g * own_rows) * before[:, :, -1] + (k[:, :, -1] * w).transpose(-1, -2) @ v[:, :, -1]
    return o.view(B, H, N * C, D)[:, :, :L], state


def _plain_attn(s):
    case, typ, scale, g = s["case"], s["q"].dtype, s["scale"], s["log_decay"]
    q, k, v = (s[n].float().transpose(1, 2) for n in ("q", "k", "v"))
    o, state = _attend(q, k, v, g, s["state"], True)

    def rounded(x):
        return x.transpose(1, 2).to(typ)

    out = {"o": rounded(scale * o), "state": state}
    if case["kind"] == "attn":
        return out
    do = s["do"].float().transpose(1, 2) * scale
    first, dlast = s["state"], s["dstate"]
    dq, _ = _attend(do, v, k, g, first.transpose(-1, -2) if first is not None else None, False)
    # backwards in time: the state's gradient behind the last token reaches it undecayed
    keep = torch.exp(g)[:, None, None]
    rev = [x.flip(2) for x in (q, k, v, do)]
    later = dlast / keep if dlast is not None else None
    dv, dstate = _attend(rev[1], rev[0], rev[3], g, later, True)
    dk, _ = _attend(rev[2], rev[3], rev[0], g, later.transpose(-1, -2) if later is not None else None, False)
    return out | {"dq": rounded(dq), "dk": rounded(dk.flip(2)), "dv": rounded(dv.flip(2)),
                  "dstate": keep * dstate if case["state"] else None}


def _plain_embed(s):
    w, ids = s["weight"], s["ids"]
    out = {"y": (s["scale"] * w[ids].float()).to(w.dtype)}
    if s["case"]["kind"] == "embed_train":
        dw = torch.zeros(w.shape, device=w.device).index_add_(0, ids, s["dy"].float())
        out["dweight"] = (s["scale"] * dw).to(w.dtype)
    return out


def _plain_clip(s):
    squares = torch.stack([x.float().square().sum(dtype=torch.float64) for x in s["grads"]])
    norm = squares.sum().sqrt()
    by = (s["max_norm"] / (norm + 1e-6)).clamp(max=1.0).float()
    clipped = [(x.float() * by).to(x.dtype).reshape(-1) for x in s["grads"]]
    flat = [torch.cat([x for x in clipped if x.dtype == f.dtype]) for f in s["flat_outs"]]
    return {"norm": norm.float(), "clipped": flat}


# ------------------------------------------------------------------------------- the definitions in 64 bits
def exact(case, seed):
    kind = case["kind"]
    if kind.startswith("attn") and case.get("L", 1) * (2 if kind == "attn_train" else 1) > 70000:
        return None
    s = prepare(case, seed)
    with torch.no_grad():
        if kind == "clip":
            return _exact_clip(s)
        return _exact_embed(s) if kind.startswith("embed") else _exact_attn(s)


def _exact_attn(s):
    """One token after another, as the recurrence and its reverse are written."""
    case = s["case"]
    step, train = case["kind"] == "attn_step", case["kind"] == "attn_train"
    # [L, B, H, D]
    q, k, v = ((s[n].double().unsqueeze(0) if step else s[n].double().permute(1, 0, 2, 3).contiguous()) for n in ("q", "k", "v"))
    keep = s["log_decay"].double().exp().view(1, -1, 1, 1)
    L, B, H, D = q.shape
    S = s["state"].double() if s["state"] is not None else torch.zeros(B, H, D, D, dtype=torch.float64, device=q.device)
    do = s["do"].double().permute(1, 0, 2, 3).contiguous() * s["scale"] if train else None
    o = torch.empty_like(q)
    dq = torch.empty_like(q) if train else None
    for t in range(L):
        S = torch.addcmul(keep * S, k[t].unsqueeze(-1), v[t].unsqueeze(-2))
        torch.matmul(q[t].unsqueeze(-2), S, out=o[t].unsqueeze(-2))
        if train:
            torch.matmul(S, do[t].unsqueeze(-1), out=dq[t].unsqueeze(-1))
    o *= s["scale"]
    if step:
        return {"o": o[0], "state": S}

    def by_batch(x):
        return x.permute(1, 0, 2, 3)

    out = {"o": by_batch(o), "state": S}
    if not train:
        return out
    G = s["dstate"].double() if s["dstate"] is not None else torch.zeros_like(S)
    dk, dv = torch.empty_like(q), torch.empty_like(q)
    for t in range(L - 1, -1, -1):  # G: the gradient of the state after token t
        G = torch.addcmul(G, q[t].unsqueeze(-1), do[t].unsqueeze(-2))
        torch.matmul(G, v[t].unsqueeze(-1), out=dk[t].unsqueeze(-1))
        torch.matmul(k[t].unsqueeze(-2), G, out=dv[t].unsqueeze(-2))
        G = keep * G
    return out | {"dq": by_batch(dq), "dk": by_batch(dk), "dv": by_batch(dv), "dstate": G if case["state"] else None}


def _exact_embed(s):
    ids, w, scale = s["ids"], s["weight"].double(), s["scale"]
    out = {"y": torch.index_select(w, 0, ids) * scale}
    if s["case"]["kind"] == "embed_train":
        # tokens sorted by id; a row's sum is the difference of two running sums
        order = torch.argsort(ids, stable=True)
        run_sum = torch.cumsum(s["dy"].double()[order], 0)
        run_sum = torch.cat([torch.zeros_like(run_sum[:1]), run_sum])
        ends = torch.searchsorted(ids[order], torch.arange(w.shape[0], device=ids.device), right=True)
        total = run_sum[ends]
        out["dweight"] = scale * torch.diff(total, dim=0, prepend=torch.zeros_like(total[:1]))
    return out


def _exact_clip(s):
    norm = math.sqrt(sum(float(torch.linalg.vector_norm(x.double())) ** 2 for x in s["grads"]))
    by = min(1.0, s["max_norm"] / (norm + 1e-6))
    types = [f.dtype for f in s["flat_outs"]]
    flat = [torch.cat([x.reshape(-1) for x in s["grads"] if x.dtype == t]).double() * by for t in types]
    return {"norm": torch.tensor(norm, dtype=torch.float64, device=s["grads"][0].device), "clipped": flat}


# ------------------------------------------------------------------------------- work
def work(case):
    kind = case["kind"]
    if kind == "clip":
        matrices, vectors = (sum(math.prod(x) for x in v) for v in _shapes(case))
        n = matrices + vectors
        size = {"bf16": 2 * n, "f32": 4 * n, "mixed": 2 * matrices + 4 * vectors}[case["dtype"]]
        return {"bytes": 2 * size + 4, "flops": 3 * n}
    es = 2 if case["dtype"] == "bf16" else 4
    if kind.startswith("embed"):
        N, V, D = case["N"], case["V"], case["D"]
        # the rows that are looked up, each read once: the expected number of different ids
        if case["ids"] == "zipf":
            share = 1.0 / (torch.arange(V, dtype=torch.float64) + 2.7)
            rows = float((1 - (1 - share / share.sum()) ** N).sum())
        else:
            rows = V * (1 - (1 - 1 / V) ** (N * (0.67 if case["ids"] == "padded" else 1.0)))
        b = 8 * N + N * D * es + rows * D * es
        if kind == "embed":
            return {"bytes": b, "flops": N * D}
        # dy read, every row of the gradient written
        return {"bytes": b + N * D * es + V * D * es, "flops": 2 * N * D}
    B, H, D = case["B"], case["H"], case["D"]
    if kind == "attn_step":
        return {"bytes": B * H * (4 * D * es + 8 * D * D), "flops": 5 * B * H * D * D}
    n = B * case["L"] * H * D
    state = 4 * B * H * D * D
    # a token's outer product and its product with the state, as the recurrence is written
    if kind == "attn":
        return {"bytes": 4 * n * es + state * (2 if case["state"] else 1), "flops": 5 * n * D}
    # q, k, v and do read, o, dq, dk and dv written
    return {"bytes": 8 * n * es + state * (4 if case["state"] else 1), "flops": 17 * n * D}
