"""Group norm with an activation, channels last (forward, gradient) against its definition in
64 bits, from one position to many, at odd group widths, strides and offsets.  Tolerances: the
derived bounds of recurrent_ref."""
import pytest
import torch

from hdcmamba_b200 import ops, recurrent
from recurrent_ref import check, norm_ref, norm_values

pytestmark = pytest.mark.gpu
DEV = "cuda"
F32, BF16 = torch.float32, torch.bfloat16


def rand(*shape, seed, dtype=F32):
    return torch.randn(*shape, generator=torch.Generator(device=DEV).manual_seed(seed), device=DEV).to(dtype)


def inputs(N, S, C, dtype, p_dtype=None, offset=0.3, scale=1.0):
    p_dtype = p_dtype or dtype
    x = (rand(N, S, C, seed=1) * scale + offset * rand(C, seed=2)).to(dtype)
    return x, (1 + 0.2 * rand(C, seed=3)).to(p_dtype), (0.3 * rand(C, seed=4)).to(p_dtype)


def run_all(x, G, w, b, act, eps=1e-5, dy=None):
    N, S, C = x.shape
    dy = rand(N, S, C, seed=5, dtype=x.dtype) if dy is None else dy
    y, mean, rstd = ops.group_norm_act(x, G, w, b, eps=eps, act=act, stats=True)
    dx, dw, db = ops.group_norm_act_bwd(dy, x, mean, rstd, G, w, b, act=act)
    ref = norm_ref(x, G, w, b, eps, act, dy)
    got = {"y": y, "mean": mean, "dx": dx}
    if w is not None:
        got["dw"] = dw
    if b is not None:
        got["db"] = db
    for k, v in got.items():
        check(v, ref[k], k)
    assert torch.equal(ops.group_norm_act(x, G, w, b, eps=eps, act=act), y)
    return got


SHAPES = [
    # one position: heads of 64, 32, 10, 7 channels, one channel, one group
    (1, 1, 64, 1), (5, 1, 768, 12), (300, 1, 1024, 16), (257, 1, 96, 3), (33, 1, 70, 7), (9, 1, 21, 3), (3, 1, 8, 8),
    (7, 1, 2048, 1), (2, 1, 4104, 2),
    # few and many positions
    (2, 2, 32, 4), (3, 5, 64, 8), (4, 16, 30, 3), (2, 49, 320, 32), (1, 64, 1, 1), (3, 77, 10, 2), (2, 225, 96, 8),
    (1, 1000, 640, 32), (2, 4096, 40, 4), (1, 5000, 33, 11), (1, 20000, 64, 2), (6, 300, 256, 1), (40, 130, 128, 32),
    # groups too wide for one CTA's channels, and at the limits of the lanes of one position
    (2, 3, 10000, 2), (3, 1, 5000, 1), (3, 1, 256, 1), (3, 1, 257, 1), (3, 1, 1024, 1), (5, 1, 1032, 1), (4, 1, 255, 1),
    (3, 10, 1500, 1), (2, 33, 2049, 3),
]


@pytest.mark.parametrize("act", ["silu", "none"])
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("N,S,C,G", SHAPES)
def test_shapes(N, S, C, G, dtype, act):
    x, w, b = inputs(N, S, C, dtype)
    run_all(x, G, w, b, act)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("with_w,with_b", [(False, False), (True, False), (False, True)])
@pytest.mark.parametrize("N,S", [(20, 1), (2, 100)])
def test_without_parameters(dtype, with_w, with_b, N, S):
    x, w, b = inputs(N, S, 48, dtype)
    run_all(x, 4, w if with_w else None, b if with_b else None, "silu")


@pytest.mark.parametrize("dtype,p_dtype", [(BF16, F32), (F32, BF16)])
@pytest.mark.parametrize("N,S", [(20, 1), (2, 300)])
def test_parameter_type(dtype, p_dtype, N, S):
    x, w, b = inputs(N, S, 64, dtype, p_dtype)
    got = run_all(x, 8, w, b, "silu")
    assert got["dw"].dtype == got["db"].dtype == p_dtype


@pytest.mark.parametrize("N,S,C,G", [(30, 1, 128, 2), (2, 500, 64, 8)])
@pytest.mark.parametrize("offset", [30.0, 1000.0])
def test_large_mean(N, S, C, G, offset):
    """The variance does not cancel: mean 1000 times the spread."""
    x = rand(N, S, C, seed=1) + offset
    w, b = 1 + 0.2 * rand(C, seed=3), 0.3 * rand(C, seed=4)
    run_all(x, G, w, b, "silu")


def test_outlier_first():
    """A first value far from all others (a poor choice of shift) costs no accuracy."""
    x = rand(2, 3000, 32, seed=1)
    x[:, 0, 0] = 1e4
    ref = norm_ref(x, 4, None, None, 1e-5, "none")
    y = ops.group_norm_act(x, 4)
    check(y, ref["y"], "y")


@pytest.mark.parametrize("N,S,C,G", [(8, 1, 64, 4), (2, 300, 32, 4), (1, 3000, 64, 8)])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_constant_groups(N, S, C, G, dtype):
    """No spread at all: rstd = 1/sqrt(eps), xh = 0, finite everywhere."""
    x = torch.full((N, S, C), 0.75, device=DEV, dtype=dtype)
    _, w, b = inputs(N, S, C, dtype)
    y, mean, rstd = ops.group_norm_act(x, G, w, b, act="none", stats=True)
    assert torch.equal(y, b.expand_as(y))
    assert torch.equal(mean, torch.full_like(mean, 0.75))
    torch.testing.assert_close(rstd, torch.full_like(rstd, 1e-5 ** -0.5), rtol=1e-5, atol=0)
    dx, dw, db = ops.group_norm_act_bwd(rand(N, S, C, seed=5, dtype=dtype), x, mean, rstd, G, w, b, act="none")
    assert bool(torch.isfinite(dx).all()) and bool((dw == 0).all())


@pytest.mark.parametrize("N,S,C,G", [(6, 1, 64, 4), (3, 300, 32, 4)])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_nan_stays_in_its_group(N, S, C, G, bad):
    x, w, b = inputs(N, S, C, F32)
    y0 = ops.group_norm_act(x, G, w, b, act="silu")
    x[1, S // 2, 0] = bad
    y = ops.group_norm_act(x, G, w, b, act="silu")
    cg = C // G
    assert bool(y[1, :, :cg].isnan().any())
    y[1, :, :cg] = y0[1, :, :cg]
    assert torch.equal(y, y0)


@pytest.mark.parametrize("scale", [1e-4, 1e3])
def test_activation_range(scale):
    """Weights that drive SiLU far into both tails, and spreads near eps."""
    N, S, C, G = 4, 60, 64, 4
    x, w, b = inputs(N, S, C, F32, scale=scale, offset=0.0)
    run_all(x, G, 30 * w, 20 * b, "silu")


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_strides(dtype):
    """Channel slices, position and sample strides, misaligned bases, NCHW tensors in channels-last
    memory and more than one position axis."""
    N, S, C, G = 3, 50, 64, 8
    buf = rand(N, S + 2, C + 17, seed=1, dtype=dtype)
    _, w, b = inputs(N, S, C, dtype)
    for off in (0, 1, 8):
        x = buf[:, 1:S + 1, off:off + C]
        got = run_all(x, G, w, b, "silu")
        again = run_all(x.contiguous(), G, w, b, "silu")
        for k in got:
            assert torch.equal(got[k], again[k]), (off, k)
    dy = rand(N, S, C + 5, seed=6, dtype=dtype)[..., 3:3 + C]
    run_all(buf[:, :S, :C], G, w, b, "silu", dy=dy)
    rows = rand(7, 2 * C + 3, seed=9, dtype=dtype)
    run_all(rows[:, C + 1:2 * C + 1].unsqueeze(1), G, w, b, "silu")
    y2 = ops.group_norm_act(rows[:, C + 1:2 * C + 1], G, w, b, act="silu")
    assert y2.shape == (7, C)
    img = rand(2, C, 6, 5, seed=8, dtype=dtype).to(memory_format=torch.channels_last).permute(0, 2, 3, 1)
    y4 = ops.group_norm_act(img, G, w, b, act="silu")
    assert y4.shape == img.shape
    assert torch.equal(y4.reshape(2, 30, C), ops.group_norm_act(img.reshape(2, 30, C), G, w, b, act="silu"))
    check(y4.reshape(2, 30, C), norm_ref(img.reshape(2, 30, C), G, w, b, 1e-5, "silu")["y"], "4-D")


@pytest.mark.parametrize("shape", [(0, 4, 32), (3, 0, 32), (0, 32)])
def test_empty(shape):
    x = torch.empty(shape, device=DEV)
    w, b = torch.ones(32, device=DEV), torch.zeros(32, device=DEV)
    y, mean, rstd = ops.group_norm_act(x, 4, w, b, act="silu", stats=True)
    assert y.shape == x.shape
    dx, dw, db = ops.group_norm_act_bwd(y, x, mean, rstd, 4, w, b, act="silu")
    assert dx.shape == x.shape and bool((dw == 0).all()) and bool((db == 0).all())


@pytest.mark.parametrize("N,S,C,G", [(3000, 1, 768, 12), (3, 5000, 96, 8), (2, 300, 256, 32)])
def test_repeats_bit_for_bit(N, S, C, G):
    x, w, b = inputs(N, S, C, BF16)
    dy = rand(N, S, C, seed=5, dtype=BF16)
    first = None
    for _ in range(4):
        y, mean, rstd = ops.group_norm_act(x, G, w, b, act="silu", stats=True)
        now = (y, mean, rstd, *ops.group_norm_act_bwd(dy, x, mean, rstd, G, w, b, act="silu"))
        if first is not None:
            assert all(torch.equal(p, q) for p, q in zip(first, now))
        first = now


def test_stream_and_graph():
    x, w, b = inputs(2, 900, 64, BF16)
    dy = rand(2, 900, 64, seed=5, dtype=BF16)
    want, mean, rstd = ops.group_norm_act(x, 8, w, b, act="silu", stats=True)
    grads = ops.group_norm_act_bwd(dy, x, mean, rstd, 8, w, b, act="silu")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = ops.group_norm_act(x, 8, w, b, act="silu")
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y, m, r = ops.group_norm_act(x, 8, w, b, act="silu", stats=True)
        dx, dw, db = ops.group_norm_act_bwd(dy, x, m, r, 8, w, b, act="silu")
    for _ in range(3):
        y.zero_(), dx.zero_(), dw.zero_()
        graph.replay()
        assert torch.equal(y, want) and torch.equal(dx, grads[0])
        assert torch.equal(dw, grads[1]) and torch.equal(db, grads[2])


@pytest.mark.parametrize("one", [True, False])
def test_offsets_beyond_32_bits(one):
    """More than 2^31 elements, as single positions and as one long sample's neighbours."""
    C, G = 512, 8
    rows = 2 ** 31 // C + 1024
    shape = (rows, 1, C) if one else (2, rows // 2, C)
    x = torch.empty(shape, device=DEV, dtype=BF16)
    x.normal_(generator=torch.Generator(device=DEV).manual_seed(1))
    w, b = (1 + 0.2 * rand(C, seed=3)).bfloat16(), (0.3 * rand(C, seed=4)).bfloat16()
    y, mean, rstd = ops.group_norm_act(x, G, w, b, act="silu", stats=True)
    dx, dw, _ = ops.group_norm_act_bwd(x, x, mean, rstd, G, w, b, act="silu")
    if one:
        ref = norm_ref(x[-500:], G, w, b, 1e-5, "silu", x[-500:])
        check(y[-500:], ref["y"], "y")
        check(dx[-500:], ref["dx"], "dx")
    else:
        for k in range(2):
            xg = x[k, :, -C // G:].double()
            m, v = xg.mean(), xg.var(correction=0)
            torch.testing.assert_close(mean[k, -1].double(), m, rtol=0, atol=1e-5)
            torch.testing.assert_close(rstd[k, -1].double(), (v + 1e-5).rsqrt(), rtol=1e-4, atol=0)
            z = (xg[-500:] - m) * (v + 1e-5).rsqrt() * w[-C // G:].double() + b[-C // G:].double()
            torch.testing.assert_close(y[k, -500:, -C // G:].double(), z * torch.sigmoid(z), rtol=2 ** -7, atol=1e-3)


# ------------------------------------------------------------------ autograd
@pytest.mark.parametrize("act", ["silu", "none"])
@pytest.mark.parametrize("N,S,C,G", [(6, 1, 24, 3), (2, 40, 20, 4)])
def test_gradient_against_differences(N, S, C, G, act):
    """Directional derivatives of the definition by central differences in 64 bits (step 1e-6);
    the fp32 gradient's own rounding, 1e-5 of the terms' size, decides."""
    x, w, b = inputs(N, S, C, F32)
    dy = rand(N, S, C, seed=5)
    leaves = [t.clone().requires_grad_() for t in (x, w, b)]
    grads = torch.autograd.grad([recurrent.group_norm_act(leaves[0], G, leaves[1], leaves[2], act=act)], leaves, [dy])

    def loss(*p):
        return float((norm_values(p[0], G, p[1], p[2], 1e-5, act) * dy.double()).sum())

    base = [t.double() for t in (x, w, b)]
    for i, gr in enumerate(grads):
        for seed in range(3):
            v = rand(*gr.shape, seed=100 + seed).double()
            up, down = list(base), list(base)
            up[i], down[i] = base[i] + 1e-6 * v, base[i] - 1e-6 * v
            want = (loss(*up) - loss(*down)) / 2e-6
            size = float((gr.double() * v).abs().sum())
            assert abs(float((gr.double() * v).sum()) - want) <= 1e-5 * size + 1e-6, (i, seed)


def test_autograd_expanded_gradient():
    """The gradient of a sum arrives expanded (stride 0)."""
    x, w, b = inputs(3, 20, 32, F32)
    x.requires_grad_()
    dx, = torch.autograd.grad(recurrent.group_norm_act(x, 4, w, b, act="silu").sum(), x)
    check(dx, norm_ref(x.detach(), 4, w, b, 1e-5, "silu", torch.ones_like(x))["dx"], "dx")


# ------------------------------------------------------------------ refusals
def test_refusals():
    x, w, b = inputs(2, 5, 32, F32)
    with pytest.raises(ValueError, match="groups"):
        ops.group_norm_act(x, 5, w, b)
    with pytest.raises(ValueError, match="groups"):
        ops.group_norm_act(x, 0, w, b)
    with pytest.raises(ValueError, match="weight"):
        ops.group_norm_act(x, 4, w[:31], b)
    with pytest.raises(ValueError, match="act"):
        ops.group_norm_act(x, 4, w, b, act="gelu")
    with pytest.raises(TypeError, match="dtype"):
        ops.group_norm_act(x.half(), 4, w, b)
    with pytest.raises(TypeError, match="mismatch"):
        ops.group_norm_act(x, 4, w, b.bfloat16())
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.group_norm_act(x, 4, w.cpu(), b)
    with pytest.raises(ValueError, match="N, ..., C"):
        ops.group_norm_act(w, 4)
    _, mean, rstd = ops.group_norm_act(x, 4, w, b, stats=True)
    with pytest.raises(ValueError, match="shape"):
        ops.group_norm_act_bwd(x[:, :4], x, mean, rstd, 4, w, b)
    with pytest.raises(ValueError, match="mean"):
        ops.group_norm_act_bwd(x, x, mean[:1], rstd, 4, w, b)
    with pytest.raises(TypeError, match="mismatch"):
        ops.group_norm_act_bwd(x.bfloat16(), x, mean, rstd, 4, w, b)
