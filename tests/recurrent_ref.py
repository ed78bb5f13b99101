"""The gated recurrence and the group norm with an activation in 64 bits, with bounds on the
rounding errors of a 32-bit evaluation (first order, from the same recurrences).

Bounds.  U = 2^-24 is fp32's unit roundoff.  Recurrence: each step multiplies by a decay whose
computed value is off by at most a few units (exp, softplus and two products, |d A| of order
one) and adds one rounding; K = 16 units per step covers them and the products of decays that
a split evaluation multiplies.  The error then obeys the recurrence of the absolute values,
E_t = a_t E_{t-1} + K U H_t with H the recurrence of |u|.  Gradients: the product rule on
values bounded the same way.  Sums of n terms: n U sum|.|.
Group norm: sums of depth up to 4096 whose roundings have random signs, so K = 64 units.
A result stored in bf16 adds half a unit in its last place, 2^-8 of its size.
"""
import torch

U = 2.0 ** -24
K_SCAN, K_NORM = 16, 64


def softplus(x):
    return torch.logaddexp(x, torch.zeros_like(x))


def _scan(a, u, h):
    out = torch.empty_like(u)
    for t in range(u.shape[1]):
        h = a[:, t] * h + u[:, t]
        out[:, t] = h
    return out


def _shift(v, first):
    return torch.cat([first.unsqueeze(1), v[:, :-1]], 1)


def scan_values(projs, A_log, ds, h0=None, reset=None):
    """y [B, L, ds] by the definition, in projs' own type (64 bits; differentiable)."""
    dt, x, b = projs[..., :ds], projs[..., ds:2 * ds], projs[..., 2 * ds:3 * ds]
    d = softplus(dt)
    a = torch.exp(-d * torch.exp(A_log))
    if reset is not None:
        a = torch.where(reset.bool().unsqueeze(-1), torch.zeros_like(a), a)
    u = d * b * x
    h = torch.zeros_like(u[:, 0]) if h0 is None else h0
    ys = []
    for t in range(u.shape[1]):
        h = a[:, t] * h + u[:, t]
        ys.append(h)
    return torch.stack(ys, 1)


def scan_ref(projs, A_log, ds, h0=None, reset=None, dy=None, dh_last=None):
    """{name: (value, error bound of a 32-bit evaluation)} in 64 bits."""
    p = projs.double()
    B, L = p.shape[:2]
    dt, x, b = p[..., :ds], p[..., ds:2 * ds], p[..., 2 * ds:3 * ds]
    A = -torch.exp(A_log.double())
    d = softplus(dt)
    a = torch.exp(d * A)
    if reset is not None:
        a = a * (~reset.bool()).unsqueeze(-1)
    u = d * b * x
    z = torch.zeros(B, ds, dtype=torch.float64, device=p.device)
    h0 = z if h0 is None else h0.double()
    k = K_SCAN * U
    y = _scan(a, u, h0)
    H = _scan(a, u.abs(), h0.abs())
    E = _scan(a, k * H, k * h0.abs())
    out = {"y": (y, E), "h_last": (y[:, -1], E[:, -1])}
    if dy is None:
        return out
    dy = dy.double()
    dh = z if dh_last is None else dh_last.double()
    def back(v, last):
        c = last
        out = torch.empty_like(v)
        for t in range(L - 1, -1, -1):
            out[:, t] = v[:, t] + c
            c = a[:, t] * out[:, t]
        return out, c
    g, dh0 = back(dy, dh)
    Gs, _ = back(dy.abs(), dh.abs())
    Eg, Eh0 = back(k * Gs, k * dh.abs())
    hp, Hp, Ep = _shift(y, h0), _shift(H, h0.abs()), _shift(E, k * h0.abs())
    s = g * a * hp
    S, Es = Gs * a * Hp, Eg * a * Hp + Gs * a * Ep + k * Gs * a * Hp
    sig = torch.sigmoid(dt)
    ddt = (s * A + g * b * x) * sig
    Et = (Es * A.abs() + Eg * (b * x).abs() + k * (S * A.abs() + Gs * (b * x).abs())) * sig
    dx, Ex = g * d * b, (Eg + k * Gs) * (d * b).abs()
    db, Eb = g * d * x, (Eg + k * Gs) * (d * x).abs()
    terms = s * d * A
    EA = (Es * (d * A).abs()).sum((0, 1)) + (L + B + K_SCAN) * U * (S * (d * A).abs()).sum((0, 1))
    out |= {"dprojs": (torch.cat([ddt, dx, db], -1), torch.cat([Et, Ex, Eb], -1)),
            "dA_log": (terms.sum((0, 1)), EA), "dh0": (dh0, Eh0 + k * Gs[:, 0])}
    return out


def norm_values(x, G, w, b, eps, act):
    """y of the group norm with activation, x [N, S, C], in x's own type (differentiable)."""
    N, S, C = x.shape
    xg = x.reshape(N, S, G, C // G)
    mean = xg.mean((1, 3), keepdim=True)
    var = ((xg - mean) ** 2).mean((1, 3), keepdim=True)
    z = ((xg - mean) / torch.sqrt(var + eps)).reshape(N, S, C)
    z = z if w is None else z * w
    z = z if b is None else z + b
    return z * torch.sigmoid(z) if act == "silu" else z


def norm_ref(x, G, w, b, eps, act, dy=None):
    """{name: (value, error bound of a 32-bit evaluation)} in 64 bits; x [N, S, C]."""
    N, S, C = x.shape
    x = x.double()
    k = K_NORM * U
    one = torch.ones(C, dtype=torch.float64, device=x.device)
    wd = one if w is None else w.double()
    bd = 0 * one if b is None else b.double()
    xg = x.reshape(N, S, G, C // G)

    def mean_of(v):
        return v.reshape(N, S, G, C // G).mean((1, 3), keepdim=True).expand(N, S, G, C // G).reshape(N, S, C)

    mean = xg.mean((1, 3), keepdim=True)
    var = ((xg - mean) ** 2).mean((1, 3), keepdim=True)
    rstd = (1 / torch.sqrt(var + eps)).expand(N, S, G, C // G).reshape(N, S, C)
    m = mean.expand(N, S, G, C // G).reshape(N, S, C)
    xh = (x - m) * rstd
    Em = k * (mean_of(x.abs()) + x.abs()) * rstd  # error of x - mean, scaled
    Ex = Em + xh.abs() * (k + mean_of(Em) ** 2 + mean_of(Em * xh.abs()))
    z = xh * wd + bd
    Ez = Ex * wd.abs() + 2 * U * (xh * wd).abs() + 2 * U * z.abs()
    q = torch.sigmoid(z)
    if act == "silu":
        y, Ey = z * q, 1.1 * Ez + k * z.abs() * q
    else:
        y, Ey = z, Ez
    out = {"y": (y, Ey), "mean": (mean.reshape(N, G), (k * xg.abs().mean((1, 3))))}
    if dy is None:
        return out
    dy = dy.double()
    if act == "silu":
        slope = q * (1 + z * (1 - q))
        dz, Ed = dy * slope, dy.abs() * (0.5 * Ez + k * (slope.abs() + q * (1 + z.abs() * (1 - q))))
    else:
        dz, Ed = dy, 0 * dy
    e, Ee = dz * wd, (Ed + U * dz.abs()) * wd.abs()
    me, mx = mean_of(e), mean_of(e * xh)
    Eme = mean_of(Ee) + k * mean_of(e.abs())
    Emx = mean_of(Ee * xh.abs() + e.abs() * Ex) + k * mean_of((e * xh).abs())
    dx = rstd * (e - me - xh * mx)
    Edx = rstd * (Ee + Eme + xh.abs() * Emx + Ex * mx.abs() + k * (e.abs() + me.abs() + (xh * mx).abs())) + \
        dx.abs() * (Em.mean() ** 2 + k) + rstd * mean_of(Em * xh.abs()) * (e.abs() + me.abs() + (xh * mx).abs())
    n = N * S
    Edw = (Ed * xh.abs() + dz.abs() * Ex).sum((0, 1)) + (k + min(n, 4096) * U) * (dz * xh).abs().sum((0, 1))
    Edb = Ed.sum((0, 1)) + (k + min(n, 4096) * U) * dz.abs().sum((0, 1))
    out |= {"dx": (dx, Edx), "dw": ((dz * xh).sum((0, 1)), Edw), "db": (dz.sum((0, 1)), Edb)}
    return out


def check(got, want, what=""):
    """got within the bound of ``want`` = (value, bound), plus its own rounding if bf16."""
    value, bound = want
    assert tuple(got.shape) == tuple(value.shape), (what, got.shape, value.shape)
    half = 2.0 ** -8 if got.dtype == torch.bfloat16 else U
    # 1e-30: below any normal result, for values that are zero by definition
    tol = bound + half * (value.abs() + bound) + 1e-30
    off = (got.double().to(value.device) - value).abs()
    bad = ~(off <= tol)
    if bool(bad.any()):
        i = int((off / tol).nan_to_num(float("inf")).argmax())
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.numel()} off; worst at {i}: got "
                             f"{float(got.reshape(-1)[i])}, want {float(value.reshape(-1)[i])} +- "
                             f"{float(tol.reshape(-1)[i])}")
