"""Linear attention with a decay for each head against its recurrence in 64 bits (bounds: attn_ref.py)."""
import pytest
import torch

from attn_ref import check_forward, check_gradient, recur
from hdcmamba_b200 import _lib, ops, recurrent

pytestmark = pytest.mark.gpu
F32, BF16 = torch.float32, torch.bfloat16


def make(dtype, B, L, H, D, state=False, seed=0, decay=None):
    g = torch.Generator().manual_seed(seed)
    q, k, v, do = (torch.randn(B, L, H, D, generator=g).to(dtype).cuda() for _ in range(4))
    ld = -torch.exp(torch.empty(H).uniform_(-7.5, -0.7, generator=g)) if decay is None else torch.full((H,), float(decay))
    s = torch.randn(B, H, D, D, generator=g).cuda() if state else None
    ds = torch.randn(B, H, D, D, generator=g).cuda() if state else None
    return q, k, v, ld.cuda(), s, do, ds


LENGTHS = [1, 2, 15, 16, 17, 63, 64, 65, 127, 129, 257]
SIZES = [1, 3, 8, 16, 20, 32, 33, 40, 64, 65, 80, 96, 100, 128]


def both(q, k, v, ld, s, do, ds, scale=0.3):
    """Forward and gradient, checked."""
    bf16 = q.dtype == BF16
    leaves = [x.detach().requires_grad_() for x in (q, k, v)] + ([s.detach().requires_grad_()] if s is not None else [])
    o, after = recurrent.decay_attention(*leaves[:3], ld, scale, leaves[3] if s is not None else None)
    check_forward(o, after, q, k, v, ld, scale, s, bf16)
    outs, douts = ([o, after], [do, ds]) if ds is not None else ([o], [do])
    grads = torch.autograd.grad(outs, leaves, douts)
    check_gradient(list(grads) + [None] * (4 - len(grads)), q, k, v, ld, scale, s, do, ds, bf16)
    return o, after, grads


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("L", LENGTHS)
def test_lengths(dtype, L):
    both(*make(dtype, 2, L, 3, 64, state=L % 2 == 1, seed=L))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("D", SIZES)
def test_head_sizes(dtype, D):
    both(*make(dtype, 2, 150, 2, D, state=True, seed=D))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("B,L,H,D", [(1, 1000, 1, 64), (1, 2049, 2, 32), (3, 700, 5, 24), (1, 640, 3, 128), (30, 200, 16, 16), (2, 1025, 20, 64), (1, 4000, 9, 40),
                                     (1, 1, 1, 1), (500, 3, 1, 8)])
def test_segments(dtype, B, L, H, D):
    """Sequences cut into several segments, the last one short, and more heads than CTAs."""
    both(*make(dtype, B, L, H, D, state=True, seed=L + D))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("decay", [0.0, -1e-4, -3.0, -40.0, -200.0, float("-inf")])
def test_decays(dtype, decay):
    """Heads that forget nothing, and heads that remember nothing; one segment and several, of both chunk lengths."""
    for L in (200, 500, 2060) if dtype == BF16 else (200,):
        q, k, v, ld, s, do, ds = make(dtype, 1, L, 2, 64, state=True, seed=5, decay=decay)
        both(q, k, v, ld, s, do, ds)


def test_each_head_has_its_own_decay():
    q, k, v, _, s, do, ds = make(BF16, 1, 300, 4, 64, state=True, seed=6)
    both(q, k, v, torch.tensor([0.0, -0.01, -1.0, -60.0]).cuda(), s, do, ds)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("D", [64, 40, 30])
def test_views(dtype, D):
    """Slices of one projection, at offsets that 16-byte loads do not allow, permuted and expanded tensors."""
    B, L, H = 2, 130, 4
    g = torch.Generator().manual_seed(7)
    ld = torch.tensor([-0.01, -0.1, -0.5, -0.02]).cuda()
    do = torch.randn(B, L, H, D, generator=g).to(dtype).cuda()
    for lead in (0, 8, 2, 1):
        proj = torch.randn(B, L, lead + 3 * H * D + 5, generator=g).to(dtype).cuda()
        q, k, v = (proj[..., lead + i * H * D:lead + (i + 1) * H * D].unflatten(-1, (H, D)) for i in range(3))
        both(q, k, v, ld, None, do, None)
    q, k, v = (torch.randn(B, H, L, D, generator=g).to(dtype).cuda().transpose(1, 2) for _ in range(3))
    both(q, k, v, ld, None, do.transpose(1, 2).contiguous().transpose(1, 2), None)
    # one head of k and v for all of q's
    k, v = (torch.randn(B, L, 1, D, generator=g).to(dtype).cuda().requires_grad_() for _ in range(2))
    q = q.detach().requires_grad_()
    o, _ = recurrent.decay_attention(q, k.expand(B, L, H, D), v.expand(B, L, H, D), ld)
    check_forward(o, ops.decay_attention(q, k.expand(B, L, H, D), v.expand(B, L, H, D), ld)[1], q, k.expand(B, L, H, D),
                  v.expand(B, L, H, D), ld, 1.0, None, dtype == BF16)
    dk, dv = torch.autograd.grad(o, [k, v], do)
    heads = [x.detach().expand(B, L, H, D).contiguous().requires_grad_() for x in (k, v)]
    o2, _ = recurrent.decay_attention(q.detach(), *heads, ld)
    per = torch.autograd.grad(o2, heads, do)
    for a, b in zip((dk, dv), per):
        tol = 2 ** -8 if dtype == BF16 else 2 ** -22  # the sum of four heads, rounded once
        assert (a.double() - b.double().sum(2, keepdim=True)).abs().max() <= tol * b.double().abs().sum(2).max()
    # a gradient that is an expanded scalar
    o3, _ = recurrent.decay_attention(q, k.expand(B, L, H, D), v.expand(B, L, H, D), ld)
    (dq,) = torch.autograd.grad(o3.sum(), [q])
    o4, _ = recurrent.decay_attention(q, k.expand(B, L, H, D), v.expand(B, L, H, D), ld)
    (dq2,) = torch.autograd.grad(o4, [q], torch.ones_like(o4))
    assert torch.equal(dq, dq2)


@pytest.mark.parametrize("D", [40, 48, 56, 64])
@pytest.mark.parametrize("L", [449, 1100, 2050, 2176])
def test_long_views(D, L):
    """Several segments, from 2048 tokens on of 128-token chunks: slices of a projection, permuted tensors, shared heads, an output view."""
    B, H = (1, 4) if L < 2000 else (2, 2)
    g = torch.Generator().manual_seed(L + D)
    ld = torch.tensor([-0.002, -0.7, -0.1, -0.02][:H]).cuda()
    do = torch.randn(B, L, H, D, generator=g).to(BF16).cuda()
    s, ds = (torch.randn(B, H, D, D, generator=g).cuda() for _ in range(2))
    proj = torch.randn(B, L, 8 + 3 * H * D, generator=g).to(BF16).cuda()
    q, k, v = (proj[..., 8 + i * H * D:8 + (i + 1) * H * D].unflatten(-1, (H, D)) for i in range(3))
    both(q, k, v, ld, s, do, ds)
    q, k, v = (torch.randn(B, H, L, D, generator=g).to(BF16).cuda().transpose(1, 2) for _ in range(3))
    both(q, k, v, ld, None, do.transpose(1, 2).contiguous().transpose(1, 2), None)
    one = torch.randn(B, L, 1, D, generator=g).to(BF16).cuda().expand(B, L, H, D)
    o, e = ops.decay_attention(q, one, v, ld, 0.3)
    check_forward(o, e, q, one, v, ld, 0.3, None, True)
    buf = torch.full((B, L + 20, H, D + 16), 7.0, device="cuda", dtype=BF16)
    for lead in (8, 4):  # 16-byte stores and single ones
        o2, _ = ops.decay_attention(q, k, v, ld, 0.3, out=buf[:, 10:10 + L, :, lead:lead + D])
        assert torch.equal(o2, ops.decay_attention(q, k, v, ld, 0.3)[0])
        o2.fill_(7)
        assert (buf == 7).all()


def test_out_view_leaves_the_rest():
    q, k, v, ld, s, _, _ = make(BF16, 2, 70, 3, 40)
    buf = torch.full((2, 90, 3, 48), 7.0, device="cuda", dtype=BF16)
    o, _ = ops.decay_attention(q, k, v, ld, out=buf[:, 10:80, :, 4:44])
    assert torch.equal(o, ops.decay_attention(q, k, v, ld)[0])
    rest = torch.ones_like(buf, dtype=torch.bool)
    rest[:, 10:80, :, 4:44] = False
    assert (buf[rest] == 7).all()


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("B,H,D", [(1, 12, 64), (3, 2, 128), (2, 3, 37), (5, 1, 1), (70, 16, 32), (2, 2, 100)])
def test_step(dtype, B, H, D):
    """A token at a time, in place and not, against the recurrence; views of a projection."""
    q, k, v, ld, s, _, _ = make(dtype, B, 4, H, D, state=True, seed=D)
    s = s.contiguous()
    S = s.clone()
    os = []
    for t in range(4):
        if t % 2:
            nxt = torch.empty_like(S)
            o, got = ops.decay_attention_step(q[:, t], k[:, t], v[:, t], ld, S, 0.3, state_out=nxt)
            assert got is nxt
            S = nxt
        else:
            o, got = ops.decay_attention_step(q[:, t], k[:, t], v[:, t], ld, S, 0.3)
            assert got is S
        os.append(o)
    ref, RS = recur(*(x.double().cpu() for x in (q, k, v, ld)), 0.3, s.double().cpu())
    check_forward(torch.stack(os, 1), S, q, k, v, ld, 0.3, s, dtype == BF16)


def test_step_at_no_decay_and_all_decay():
    q, k, v, _, s, _, _ = make(F32, 2, 1, 2, 16, state=True)
    ld = torch.tensor([0.0, float("-inf")]).cuda()
    o, S = ops.decay_attention_step(q[:, 0], k[:, 0], v[:, 0], ld, s.clone())
    kv = k[:, 0, :, :, None] * v[:, 0, :, None, :]
    assert torch.allclose(S[:, 0], s[:, 0] + kv[:, 0], rtol=1e-6, atol=1e-6) and torch.equal(S[:, 1], kv[:, 1])


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_windows_and_steps_continue_a_sequence(dtype):
    """Two windows, and then steps, against one sequence; the state's gradient joins the windows."""
    q, k, v, ld, s, do, ds = make(dtype, 2, 190, 3, 48, state=True, seed=9)
    bf16 = dtype == BF16
    ql, kl, vl = (x.detach().requires_grad_() for x in (q, k, v))
    o1, m = recurrent.decay_attention(ql[:, :77], kl[:, :77], vl[:, :77], ld, 0.3, s)
    o2, e = recurrent.decay_attention(ql[:, 77:], kl[:, 77:], vl[:, 77:], ld, 0.3, m)
    check_forward(torch.cat([o1, o2], 1), e, q, k, v, ld, 0.3, s, bf16)
    grads = torch.autograd.grad([o1, o2, e], [ql, kl, vl], [do[:, :77].contiguous(), do[:, 77:].contiguous(), ds])
    check_gradient(list(grads) + [None], q, k, v, ld, 0.3, s, do, ds, bf16)
    o, m = ops.decay_attention(q[:, :188], k[:, :188], v[:, :188], ld, 0.3, s)
    tail = [ops.decay_attention_step(q[:, t], k[:, t], v[:, t], ld, m, 0.3)[0] for t in (188, 189)]
    check_forward(torch.cat([o, torch.stack(tail, 1)], 1), m, q, k, v, ld, 0.3, s, bf16)


def test_gradient_against_differences():
    """fp32 kernels against central differences of the recurrence in 64 bits."""
    q, k, v, ld, s, do, ds = make(F32, 1, 70, 2, 24, state=True, seed=11)
    leaves = [x.detach().requires_grad_() for x in (q, k, v, s)]
    o, e = recurrent.decay_attention(*leaves[:3], ld, 0.3, leaves[3])
    grads = torch.autograd.grad([o, e], leaves, [do, ds])
    gen = torch.Generator().manual_seed(1)
    base = [x.detach().double().cpu() for x in (q, k, v, s)]
    for i in range(4):
        d = torch.randn(base[i].shape, generator=gen, dtype=torch.float64)
        h = 1e-5

        def value(sign):
            x = list(base)
            x[i] = x[i] + sign * h * d
            oo, ee = recur(x[0], x[1], x[2], ld.double().cpu(), 0.3, x[3])
            return (oo * do.double().cpu()).sum() + (ee * ds.double().cpu()).sum()

        want = float((value(1) - value(-1)) / (2 * h))
        got = float((grads[i].double().cpu() * d).sum())
        # the values are linear or bilinear in each argument: differences are exact up to 64-bit roundings / h
        assert abs(got - want) <= 1e-4 * float((grads[i].double().cpu().abs() * d.abs()).sum()) + 1e-6


def test_unused_outputs_and_inputs():
    q, k, v, ld, s, do, ds = make(F32, 1, 40, 2, 16, state=True)
    kl = k.detach().requires_grad_()
    _, e = recurrent.decay_attention(q, kl, v, ld, 1.0, s)
    (dk,) = torch.autograd.grad(e, [kl], ds)  # o unused
    check_gradient([None, dk, None, None], q, k, v, ld, 1.0, s, torch.zeros_like(do), ds, False)
    out = recurrent.decay_attention(q, k, v, ld, 1.0, s)
    assert not out[0].requires_grad
    sb = s.to(BF16).requires_grad_()
    _, e = recurrent.decay_attention(q, k, v, ld, 1.0, sb)
    assert torch.autograd.grad(e.sum(), [sb])[0].dtype == BF16
    with pytest.raises(RuntimeError, match="differentiable once"):
        o, _ = recurrent.decay_attention(q, kl, v, ld)
        torch.autograd.grad(o.sum(), [kl], create_graph=True)


def test_empty():
    for dtype in (F32, BF16):
        q, k, v, ld, s, do, ds = make(dtype, 2, 0, 3, 16, state=True)
        sl = s.clone().requires_grad_()
        o, e = recurrent.decay_attention(q, k, v, ld, 1.0, sl)
        assert o.shape == q.shape and torch.equal(e, s)
        (d,) = torch.autograd.grad(e, [sl], ds)
        assert torch.equal(d, ds)
        o, e = ops.decay_attention(q, k, v, ld)
        assert (e == 0).all()
        q, k, v, ld, s, do, ds = make(dtype, 0, 5, 3, 16, state=True)
        assert ops.decay_attention(q, k, v, ld, state=s)[0].shape == (0, 5, 3, 16)
        assert ops.decay_attention_step(q[:, 0], k[:, 0], v[:, 0], ld, s)[0].shape == (0, 3, 16)


@pytest.mark.parametrize("L", [130, 900, 2100])
def test_same_bits_again_on_another_stream_and_from_two_graphs(L):
    q, k, v, ld, s, do, ds = make(BF16, 2, L, 4, 64, state=True, seed=13)
    leaves = [x.detach().requires_grad_() for x in (q, k, v)]

    def run():
        o, e = recurrent.decay_attention(*leaves, ld, 0.3, s)
        return [o.detach(), e.detach(), *torch.autograd.grad([o, e], leaves, [do, ds])]

    first = run()
    for a, b in zip(first, run()):
        assert torch.equal(a, b)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = run()
    torch.cuda.current_stream().wait_stream(side)
    for a, b in zip(first, other):
        assert torch.equal(a, b)
    graphs = []
    for _ in range(2):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr), torch.no_grad():
            o, e, st = ops.decay_attention(q, k, v, ld, 0.3, s, return_states=True)
            grads = ops.decay_attention_bwd(do, q, k, v, ld, st, 0.3, ds)[:3]
        graphs.append((gr, [o, e, *grads]))
    for _ in range(2):
        for gr, outs in graphs:
            for x in outs:
                x.fill_(float("nan"))
            gr.replay()
        for gr, outs in graphs:
            for a, b in zip(first, outs):
                assert torch.equal(a, b)


def test_offsets_past_32_bits():
    """Batches that lie more than 2^31 elements apart."""
    far = 2 ** 31 + 64
    buf = torch.empty(far + 70 * 2 * 64, device="cuda", dtype=BF16)
    x = buf.as_strided((2, 70, 2, 64), (far, 128, 64, 1))
    q, k, v, ld, s, do, ds = make(BF16, 2, 70, 2, 64, seed=15)
    want, _ = ops.decay_attention(q, k, v, ld)
    x.copy_(q)
    got, _ = ops.decay_attention(x, k, v, ld)
    assert torch.equal(want, got)
    x.copy_(k)
    assert torch.equal(want, ops.decay_attention(q, x, v, ld)[0])
    got, _ = ops.decay_attention(q, k, v, ld, out=x)
    assert torch.equal(want, x)


@pytest.mark.parametrize("L", [300, 2100])
def test_non_finite_tokens_stay_in_their_sequence(L):
    """Infinities and NaN of a token reach its own batch and head, from at most 127 tokens before it on (a chunk's
    tokens are computed together: zeros of the causal mask times infinity)."""
    q, k, v, ld, _, _, _ = make(BF16, 2, L, 2, 64, seed=17)
    want, _ = ops.decay_attention(q, k, v, ld)
    v[0, 200, 1, 3] = float("nan")
    k[0, 210, 1, 5] = float("inf")
    got, _ = ops.decay_attention(q, k, v, ld)
    assert torch.equal(got[1], want[1]) and torch.equal(got[0, :, 0], want[0, :, 0])
    assert torch.equal(got[0, :73, 1], want[0, :73, 1]) and torch.isnan(got[0, 200:, 1, 3]).all()


def test_the_same_tensors_again_after_a_view_that_tma_does_not_take():
    """Strides past what a tensor map holds and heads that share memory go another way, with the same roundings."""
    q, k, v, ld, _, _, _ = make(BF16, 1, 2100, 2, 64, seed=19)
    one = k[:, :, :1]
    a, ea = ops.decay_attention(q, one.expand(-1, -1, 2, -1), v, ld, 0.3)
    b, eb = ops.decay_attention(q, one.repeat(1, 1, 2, 1), v, ld, 0.3)
    assert (a.float() - b.float()).norm() <= 2 * 2 ** -8 * b.float().norm() and torch.equal(ea, eb)


def test_no_device_error():
    torch.cuda.synchronize()
    assert _lib.load().hdc_device_error(1) == 0
