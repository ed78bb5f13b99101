"""CPU tests of the gated recurrence and the group norm with an activation: the C entry points'
refusals (all before any CUDA call), CPU inputs, and the 64-bit definitions that the GPU tests
compare with, their gradients against autograd."""
import ctypes

import pytest
import torch

from hdcmamba_b200 import _lib, ops, recurrent
from recurrent_ref import norm_ref, norm_values, scan_ref, scan_values

P = ctypes.c_void_p
OK, E_DTYPE, E_SHAPE, E_ALIGN, E_NULL, E_WORKSPACE = 0, -1, -2, -3, -4, -5
BIG = 1 << 40


def scan_fwd(dtype=1, a=0, projs=16, A=16, h0=None, y=16, y_st=8, ws=16, wsb=BIG, B=2, L=4, ds=8):
    return _lib.load().hdc_gated_scan_fwd(dtype, a, P(projs), 96, 24, P(A), P(h0), None, P(y), 32, y_st, P(16), None,
                                          P(ws), wsb, B, L, ds, None)


def scan_bwd(dtype=1, a=0, projs=16, A=16, states=16, dy=16, dprojs=16, dp_st=24, dA=16, ws=16, wsb=BIG, B=2, L=4, ds=8):
    return _lib.load().hdc_gated_scan_bwd(dtype, a, P(projs), 96, 24, P(A), P(states), None, P(dy), 32, 8, None,
                                          P(dprojs), 96, dp_st, P(dA), None, P(ws), wsb, B, L, ds, None)


def step(dtype=1, a=0, projs=16, A=16, h=16, h_out=16, y=16, y_sb=8, B=2, ds=8):
    return _lib.load().hdc_gated_step(dtype, a, P(projs), 24, P(A), P(h), None, P(h_out), P(y), y_sb, B, ds, None)


def norm_fwd(dtype=1, p=1, x=16, w=16, b=16, y=16, mean=16, rstd=16, ws=16, wsb=BIG, N=2, S=3, C=8, G=2, act=1):
    return _lib.load().hdc_group_norm_fwd(dtype, p, P(x), 24, 8, P(w), P(b), P(y), 24, 8, P(mean), P(rstd), P(ws), wsb,
                                          N, S, C, G, 1e-5, act, None)


def norm_bwd(dtype=1, p=1, dy=16, x=16, mean=16, rstd=16, w=16, dx=16, dw=16, ws=16, wsb=BIG, N=2, S=3, C=8, G=2, act=1):
    return _lib.load().hdc_group_norm_bwd(dtype, p, P(dy), 24, 8, P(x), 24, 8, P(mean), P(rstd), P(w), P(16), P(dx),
                                          24, 8, P(dw), P(16), P(ws), wsb, N, S, C, G, act, None)


@pytest.mark.parametrize("call,code", [
    (lambda: scan_fwd(dtype=7), E_DTYPE), (lambda: scan_fwd(a=2), E_DTYPE), (lambda: scan_fwd(ds=0), E_SHAPE),
    (lambda: scan_fwd(L=-1), E_SHAPE), (lambda: scan_fwd(B=65536), E_SHAPE), (lambda: scan_fwd(L=1 << 31), E_SHAPE),
    (lambda: scan_fwd(projs=None), E_NULL), (lambda: scan_fwd(A=None), E_NULL), (lambda: scan_fwd(y=None), E_NULL),
    (lambda: scan_fwd(projs=17), E_ALIGN), (lambda: scan_fwd(dtype=0, y=18), E_ALIGN),
    (lambda: scan_fwd(h0=18), E_ALIGN), (lambda: scan_fwd(y_st=7), E_SHAPE), (lambda: scan_fwd(B=0), OK),
    (lambda: scan_bwd(dtype=-1), E_DTYPE), (lambda: scan_bwd(ds=-3), E_SHAPE), (lambda: scan_bwd(states=None), E_NULL),
    (lambda: scan_bwd(dA=None), E_NULL), (lambda: scan_bwd(dy=None), E_NULL), (lambda: scan_bwd(dprojs=None), E_NULL),
    (lambda: scan_bwd(dp_st=23), E_SHAPE), (lambda: scan_bwd(wsb=4), E_WORKSPACE),
    (lambda: scan_bwd(ws=None), E_WORKSPACE), (lambda: scan_bwd(states=18), E_ALIGN),
    (lambda: step(dtype=3), E_DTYPE), (lambda: step(h=None), E_NULL), (lambda: step(h_out=None), E_NULL),
    (lambda: step(y_sb=7), E_SHAPE), (lambda: step(h=18), E_ALIGN), (lambda: step(B=0), OK),
    (lambda: norm_fwd(dtype=2), E_DTYPE), (lambda: norm_fwd(p=5), E_DTYPE), (lambda: norm_fwd(G=3), E_SHAPE),
    (lambda: norm_fwd(G=0), E_SHAPE), (lambda: norm_fwd(C=0), E_SHAPE), (lambda: norm_fwd(N=-1), E_SHAPE),
    (lambda: norm_fwd(act=2), E_SHAPE), (lambda: norm_fwd(C=1 << 17, G=1), E_SHAPE),
    (lambda: norm_fwd(N=1 << 30, G=8), E_SHAPE), (lambda: norm_fwd(x=None), E_NULL),
    (lambda: norm_fwd(mean=None), E_NULL), (lambda: norm_fwd(x=17), E_ALIGN), (lambda: norm_fwd(mean=18), E_ALIGN),
    (lambda: norm_fwd(N=0), OK), (lambda: norm_fwd(S=0), OK),
    (lambda: norm_bwd(dtype=2), E_DTYPE), (lambda: norm_bwd(G=3), E_SHAPE), (lambda: norm_bwd(mean=None), E_NULL),
    (lambda: norm_bwd(dx=None), E_NULL), (lambda: norm_bwd(wsb=4), E_WORKSPACE), (lambda: norm_bwd(dw=17), E_ALIGN),
])
def test_refusals_before_any_cuda_call(call, code):
    assert call() == code
    if code:
        assert _lib.load().hdc_error_string()


def test_cpu_tensors_raise():
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.gated_scan(torch.zeros(1, 4, 24), torch.zeros(8), 8)
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.gated_step(torch.zeros(1, 24), torch.zeros(8), torch.zeros(1, 8), 8)
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.group_norm_act(torch.zeros(2, 8), 2)
    with pytest.raises(RuntimeError, match="CUDA"):
        recurrent.gated_scan(torch.zeros(1, 4, 24, requires_grad=True), torch.zeros(8), 8)
    with pytest.raises(RuntimeError, match="CUDA"):
        recurrent.GatedRecurrentBlock(16, 16, 2)(torch.zeros(1, 4, 16))
    with pytest.raises(ValueError, match="num_heads"):
        recurrent.GatedRecurrentBlock(16, 18, 4)


def test_scan_definition_against_autograd():
    g = torch.Generator().manual_seed(0)
    B, L, ds = 2, 30, 5
    p = torch.randn(B, L, 3 * ds, generator=g, dtype=torch.float64)
    A = 0.3 * torch.randn(ds, generator=g, dtype=torch.float64)
    h0, dy, dh = (torch.randn(*s, generator=g, dtype=torch.float64) for s in ((B, ds), (B, L, ds), (B, ds)))
    reset = torch.rand(B, L, generator=g) < 0.1
    leaves = [t.clone().requires_grad_() for t in (p, A, h0)]
    y = scan_values(leaves[0], leaves[1], ds, leaves[2], reset)
    want = torch.autograd.grad([y, y[:, -1]], leaves, [dy, dh])
    ref = scan_ref(p, A, ds, h0, reset, dy, dh)
    torch.testing.assert_close(ref["y"][0], y.detach(), rtol=1e-12, atol=1e-12)
    for k, w in zip(("dprojs", "dA_log", "dh0"), want):
        torch.testing.assert_close(ref[k][0], w, rtol=1e-10, atol=1e-10)
        assert bool((ref[k][1] >= 0).all())


@pytest.mark.parametrize("act", ["silu", "none"])
def test_norm_definition_against_autograd(act):
    g = torch.Generator().manual_seed(0)
    N, S, C, G = 3, 7, 12, 4
    x, w, b, dy = (torch.randn(*s, generator=g, dtype=torch.float64) for s in ((N, S, C), (C,), (C,), (N, S, C)))
    leaves = [t.clone().requires_grad_() for t in (x, w, b)]
    y = norm_values(leaves[0], G, leaves[1], leaves[2], 1e-5, act)
    want = torch.autograd.grad(y, leaves, dy)
    ref = norm_ref(x, G, w, b, 1e-5, act, dy)
    torch.testing.assert_close(ref["y"][0], y.detach(), rtol=1e-12, atol=1e-12)
    for k, v in zip(("dx", "dw", "db"), want):
        torch.testing.assert_close(ref[k][0], v, rtol=1e-9, atol=1e-9)
