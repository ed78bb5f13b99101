"""Decayed linear attention in 64 bits, by its recurrence, and how far a kernel may be from it.

Bounds.  U = 2^-24 is fp32's unit roundoff, E = 2^-8 the largest relative error of a rounding to bf16.
Let A be the value with every product replaced by its size.

* Element by element.  fp32 sums of products and decays: K = 64 units of A (sums of up to some thousand
  terms whose roundings have random signs, exp of a product, factors of a split evaluation).  bf16 tensors:
  the product of two tokens or the state is rounded to bf16 once before it multiplies (at most E A), and the
  result once (at most E |value|).
* In the 2-norm of a batch and head.  Roundings of operands have random signs, so their part is at most
  E / sqrt(3) of the value's norm; with the result's own E that stays below 2 E.  fp32: K U.
"""
import torch

U, E, K = 2.0 ** -24, 2.0 ** -8, 64


def recur(q, k, v, g, scale, state=None):
    """(o [B, L, H, D], state [B, H, D, D]) in the inputs' own type (64 bits; differentiable)."""
    B, L, H, D = q.shape
    S = torch.zeros(B, H, D, D, dtype=q.dtype) if state is None else state
    keep = torch.exp(g)[:, None, None]
    keep = torch.where(torch.isinf(g)[:, None, None], torch.zeros_like(keep), keep)
    o = []
    for t in range(L):
        S = keep * S + k[:, t, :, :, None] * v[:, t, :, None, :]
        o.append(scale * (q[:, t, :, None, :] @ S).squeeze(-2))
    return (torch.stack(o, 1) if L else q.clone()), S


def gradient(q, k, v, g, scale, state, do, dstate):
    """(dq, dk, dv, dstate before) by the reverse recurrence, in 64 bits."""
    B, L, H, D = q.shape
    S = torch.zeros(B, H, D, D, dtype=q.dtype) if state is None else state
    G = torch.zeros(B, H, D, D, dtype=q.dtype) if dstate is None else dstate
    keep = torch.exp(g)[:, None, None]
    dq, dk, dv = torch.zeros_like(q), torch.zeros_like(q), torch.zeros_like(q)
    for t in range(L):
        S = keep * S + k[:, t, :, :, None] * v[:, t, :, None, :]
        dq[:, t] = scale * (S @ do[:, t, :, :, None]).squeeze(-1)
    for t in range(L - 1, -1, -1):
        G = G + scale * q[:, t, :, :, None] * do[:, t, :, None, :]
        dk[:, t] = (G @ v[:, t, :, :, None]).squeeze(-1)
        dv[:, t] = (k[:, t, :, None, :] @ G).squeeze(-2)
        G = keep * G
    return dq, dk, dv, G


def close(name, got, ref, size, bf16):
    """got against ref (64 bits) with the bounds above; size: A.  Tensors [B, (L,) H, ...]."""
    got = got.detach().double().cpu()
    assert got.shape == ref.shape, (name, got.shape, ref.shape)
    assert torch.isfinite(got).all(), f"{name}: not finite"
    err = (got - ref).abs()
    most = K * U * size + (E * (size + ref.abs()) if bf16 else 0.0)
    bad = err > most + 1e-37
    assert not bad.any(), f"{name}: {int(bad.sum())} of {err.numel()} off, most {float((err / (most + 1e-37)).max()):.2f} of the bound"
    if ref.numel():
        h = 2 if ref.dim() == 4 and not name.endswith("state") else 1  # the head's dim
        dims = [d for d in range(ref.dim()) if d not in (0, h)]
        e, n = err.square().sum(dims).sqrt(), ref.square().sum(dims).sqrt()
        part = 2 * E if bf16 else K * U
        assert (e <= part * n + 1e-30).all(), f"{name}: norm of the error {float((e / (n + 1e-30)).max()):.3g}, bound {part:.3g}"


def check_forward(o, after, q, k, v, g, scale, state, bf16):
    a = [x.detach().double().cpu() for x in (q, k, v, g)]
    s = state.detach().double().cpu() if state is not None else None
    ref, S = recur(*a, scale, s)
    size, SA = recur(a[0].abs(), a[1].abs(), a[2].abs(), a[3], abs(scale), s.abs() if s is not None else None)
    close("o", o, ref, size, bf16)
    close("state", after, S, SA, False)


def check_gradient(grads, q, k, v, g, scale, state, do, dstate, bf16):
    a = [x.detach().double().cpu() for x in (q, k, v, g)]
    s, do, ds = (x.detach().double().cpu() if x is not None else None for x in (state, do, dstate))

    def size(x):
        return x.abs() if x is not None else None

    ref = gradient(*a, scale, s, do, ds)
    big = gradient(a[0].abs(), a[1].abs(), a[2].abs(), a[3], abs(scale), size(s), size(do), size(ds))
    for name, got, r, b in zip(("dq", "dk", "dv", "dstate"), grads, ref, big):
        if got is not None:
            close(name, got, r, b, bf16 and name != "dstate")
