"""The norm over all gradients and clipping against 64 bits.

The norm: sums of 32 squares in fp32 (at most 33 U relative, all terms positive), the rest in 64 bits, halved by the
root, and a rounding to fp32: 20 U.  A scaled element: the factor and the product, 3 U more, and a rounding to
bf16 (2^-8)."""
import math

import pytest
import torch

from hdcmamba_b200 import ops, training

pytestmark = pytest.mark.gpu
F32, BF16 = torch.float32, torch.bfloat16
U = 2.0 ** -24


def norm_of(grads):
    return math.sqrt(sum(float(g.double().square().sum()) for g in grads))


def check(before, after, norm, max_norm):
    want = norm_of(before)
    assert abs(float(norm) - want) <= 20 * U * want
    by = min(1.0, max_norm / (want + 1e-6))
    for b, a in zip(before, after):
        ref = b.double() * by
        tol = 24 * U + (2 ** -8 if a.dtype == BF16 else 0)
        assert ((a.double() - ref).abs() <= tol * ref.abs() + 1e-44).all()
        if want < 0.999 * max_norm:
            assert torch.equal(a, b)


SIZES = [1, 7, 8, 9, 15, 8191, 8192, 8193, 8200, 16385, 100000, 3, 0, 65536, 24581]


@pytest.mark.parametrize("types", ["f32", "bf16", "mixed"])
@pytest.mark.parametrize("max_norm", [0.5, 1e9])
@pytest.mark.parametrize("place", [True, False])
def test_sizes(types, max_norm, place):
    g = torch.Generator().manual_seed(1)
    grads = [torch.randn(n, generator=g).to(F32 if types == "f32" or (types == "mixed" and i % 2) else BF16).cuda()
             for i, n in enumerate(SIZES)]
    before = [x.clone() for x in grads]
    if place:
        norm = ops.clip_grads(grads, max_norm)
        check(before, grads, norm, max_norm)
    else:
        out = [torch.full_like(x, 7) for x in grads]
        norm = ops.clip_grads(grads, max_norm, out=out)
        check(before, out, norm, max_norm)
        assert all(torch.equal(a, b) for a, b in zip(before, grads))
    only = ops.clip_grads(before, None)
    assert torch.equal(only, norm)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("lead_in,lead_out", [(0, 0), (1, 1), (3, 3), (0, 1), (5, 2), (7, 0)])
def test_unaligned_views(dtype, lead_in, lead_out):
    """Tensors that lie anywhere in a buffer, and outputs at another distance from 16-byte borders."""
    g = torch.Generator().manual_seed(2)
    sizes = [20000, 13, 8192, 1, 30001]
    a = torch.randn(lead_in + sum(sizes) + 9, generator=g).to(dtype).cuda()
    b = torch.full((lead_out + sum(sizes) + 9,), 7.0, device="cuda").to(dtype)
    grads, outs, i, o = [], [], lead_in, lead_out
    for n in sizes:
        grads.append(a[i:i + n])
        outs.append(b[o:o + n])
        i, o = i + n, o + n
    keep = a.clone()
    norm = ops.clip_grads(grads, 2.0, out=outs)
    check(grads, outs, norm, 2.0)
    assert torch.equal(a, keep) and (b[:lead_out] == 7).all() and (b[o:] == 7).all()
    before = [x.clone() for x in grads]
    norm = ops.clip_grads(grads, 2.0)
    check(before, grads, norm, 2.0)
    assert torch.equal(a[:lead_in], keep[:lead_in]) and torch.equal(a[i:], keep[i:])


def test_more_tensors_than_a_launch_takes():
    g = torch.Generator().manual_seed(3)
    grads = [torch.randn(1 + i % 50, generator=g).cuda() for i in range(1300)]
    before = [x.clone() for x in grads]
    norm = ops.clip_grads(grads, 1.0)
    check(before, grads, norm, 1.0)


@pytest.mark.parametrize("size", [1e-30, 1e-20, 1e-10, 1e15, 1e19, 1e30])
def test_squares_past_fp32(size):
    """|g|^2 below and above fp32's range; zeros beside."""
    g = torch.Generator().manual_seed(4)
    for dtype in (F32, BF16):
        x = (torch.randn(30000, generator=g) * size).to(dtype).cuda()
        x[1000:9000] = 0
        norm = ops.clip_grads([x.clone()], None)
        want = norm_of([x])
        assert abs(float(norm) - want) <= 20 * U * want + 1e-44
        y = x.clone()
        n2 = ops.clip_grads([y], 1.0)
        assert torch.equal(norm, n2)
        if size >= 1e15:
            check([x], [y], norm, 1.0)
        else:
            assert torch.equal(x, y)


def test_non_finite_and_zero():
    x, y = torch.ones(100, device="cuda"), torch.ones(50, device="cuda", dtype=BF16)
    x[3] = float("inf")
    norm = ops.clip_grads([x, y], 1.0)
    assert norm == float("inf") and torch.isnan(x[3]) and (y == 0).all() and (x[4:] == 0).all()
    x, y = torch.ones(100, device="cuda"), torch.ones(50, device="cuda", dtype=BF16)
    y[7] = float("nan")
    assert torch.isnan(ops.clip_grads([x, y], 1.0)) and torch.isnan(x).all() and torch.isnan(y).all()
    z = torch.zeros(1000, device="cuda")
    assert ops.clip_grads([z], 1.0) == 0 and (z == 0).all()
    e = torch.zeros(0, device="cuda")
    assert ops.clip_grads([e, e], 1.0) == 0
    x = torch.ones(100, device="cuda")
    ops.clip_grads([x], 0.0)
    assert (x == 0).all()
    x = torch.ones(100, device="cuda")
    assert ops.clip_grads([x], float("inf")) == 10 and (x == 1).all()


def test_parameters():
    p = [torch.nn.Parameter(torch.ones(64, 33, device="cuda")), torch.nn.Parameter(torch.ones(5, device="cuda")),
         torch.nn.Parameter(torch.ones(48, 40, device="cuda", dtype=BF16))]
    g = torch.Generator().manual_seed(5)
    for dense in (True, False):
        p[0].grad = torch.randn(64, 33, generator=g).cuda() if dense else torch.randn(33, 64, generator=g).cuda().t()
        p[2].grad = torch.randn(48, 40, generator=g).to(BF16).cuda()
        before = [p[0].grad.clone(), p[2].grad.clone()]
        norm = training.clip_grad_norm_(iter(p), 3.0)
        check(before, [p[0].grad, p[2].grad], norm, 3.0)
    assert training.clip_grad_norm_([p[1]], 1.0) == 0
    norm = training.clip_grad_norm_(p[2], 0.5)
    assert p[2].grad.float().norm() < 0.51


def test_graph_replays_on_new_values():
    xs = [torch.randn(50000, device="cuda"), torch.randn(77, device="cuda").to(BF16)]
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr):
        norm = ops.clip_grads(xs, 1.0)
    for k in range(3):
        for x in xs:
            x.copy_(torch.randn(x.shape, device="cuda") * (k + 1))
        before = [x.clone() for x in xs]
        gr.replay()
        check(before, xs, norm, 1.0)
