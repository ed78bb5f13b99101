"""The gated recurrence (forward, gradient, step) against its definition in 64 bits, at the
lengths, widths, strides, resets and values where it can go wrong.  Tolerances: the derived
bounds of recurrent_ref."""
import pytest
import torch

from hdcmamba_b200 import _lib, ops, recurrent
from recurrent_ref import check, scan_ref, scan_values

pytestmark = pytest.mark.gpu
DEV = "cuda"
F32, BF16 = torch.float32, torch.bfloat16


def inputs(B, L, ds, dtype, seed=0, extra=0, pad_rows=0, shift=0):
    """(projs view, A_log): dt about the layer's initial 0.001 .. 0.1 after softplus."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    W = 3 * ds + extra
    buf = torch.randn(B, L + pad_rows, W + shift, generator=g, device=DEV)
    d0 = 0.001 + 0.099 * torch.rand(ds, generator=g, device=DEV)
    buf[..., shift:shift + ds] = torch.log(torch.expm1(d0)) + buf[..., shift:shift + ds]
    projs = buf.to(dtype)[:, :L, shift:]
    return projs, torch.log(torch.linspace(0.5, 1.5, ds, device=DEV))


def rand(*shape, seed, dtype=F32):
    return torch.randn(*shape, generator=torch.Generator(device=DEV).manual_seed(seed), device=DEV).to(dtype)


def run_all(projs, A_log, ds, h0=None, reset=None, dh=True):
    B, L = projs.shape[:2]
    dy = rand(B, L, ds, seed=7, dtype=projs.dtype)
    dhl = rand(B, ds, seed=8) if dh else None
    y, h, st = ops.gated_scan(projs, A_log, ds, h0=h0, reset=reset, return_states=True)
    dp, dA, dh0 = ops.gated_scan_bwd(dy, projs, A_log, st, ds, reset=reset, dh_last=dhl, need_dh0=True)
    ref = scan_ref(projs, A_log, ds, h0, reset, dy, dhl)
    got = {"y": y, "h_last": h, "dprojs": dp, "dA_log": dA, "dh0": dh0}
    for k, v in got.items():
        check(v, ref[k], k)
    return got


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("B,L,ds", [
    (1, 1, 1), (2, 1, 64), (1, 2, 3), (3, 7, 5), (2, 127, 64), (2, 128, 66), (1, 129, 65), (2, 255, 33), (1, 257, 192),
    (1, 1024, 16), (1, 4100, 72), (5, 300, 130), (1, 2500, 512), (70, 40, 24),
])
def test_shapes(dtype, B, L, ds):
    projs, A_log = inputs(B, L, ds, dtype)
    run_all(projs, A_log, ds, h0=rand(B, ds, seed=3))
    run_all(projs, A_log, ds, dh=False)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("extra,pad_rows,shift", [(0, 3, 0), (8, 0, 0), (5, 0, 0), (16, 2, 8), (0, 0, 1), (1, 0, 2)])
def test_strided_and_misaligned_rows(dtype, extra, pad_rows, shift):
    B, L, ds = 2, 300, 64
    projs, A_log = inputs(B, L, ds, dtype, extra=extra, pad_rows=pad_rows, shift=shift)
    got = run_all(projs, A_log, ds, h0=rand(B, ds, seed=3))
    tight = projs[..., :3 * ds].contiguous()
    again = run_all(tight, A_log, ds, h0=rand(B, ds, seed=3))
    for k in got:
        assert torch.equal(got[k], again[k]), k  # the layout does not change the arithmetic


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("off,width", [(0, 64), (8, 80), (1, 67)])
def test_output_views(dtype, off, width):
    B, L, ds = 2, 200, 64
    projs, A_log = inputs(B, L, ds, dtype)
    y0, h0 = ops.gated_scan(projs, A_log, ds)
    buf = torch.full((B, L, width), 7.0, device=DEV, dtype=dtype)
    out = buf[..., off:off + ds]
    y, h = ops.gated_scan(projs, A_log, ds, out=out)
    assert y.data_ptr() == out.data_ptr() and torch.equal(out, y0) and torch.equal(h, h0)
    rest = torch.cat([buf[..., :off], buf[..., off + ds:]], -1)
    assert bool((rest == 7.0).all())
    # gradients into the first columns of a wider buffer
    st = ops.gated_scan(projs, A_log, ds, return_states=True)[2]
    dy = rand(B, L, ds, seed=7, dtype=dtype)
    dp = ops.gated_scan_bwd(dy, projs, A_log, st, ds)[0]
    wide = torch.full((B, L, 3 * ds + width), 7.0, device=DEV, dtype=dtype)
    ops.gated_scan_bwd(dy, projs, A_log, st, ds, out=wide)
    assert torch.equal(wide[..., :3 * ds], dp) and bool((wide[..., 3 * ds:] == 7.0).all())


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("where", ["first", "every", "random", "ends", "none", "last"])
def test_resets(dtype, where):
    B, L, ds = 3, 517, 70
    projs, A_log = inputs(B, L, ds, dtype)
    r = torch.zeros(B, L, dtype=torch.bool, device=DEV)
    if where == "first":
        r[:, 0] = True
    elif where == "every":
        r[:] = True
    elif where == "random":
        r[:] = torch.rand(B, L, generator=torch.Generator(device=DEV).manual_seed(5), device=DEV) < 0.02
    elif where == "ends":
        r[:, 127::128] = True
        r[:, 128::128] = True
    elif where == "last":
        r[:, -1] = True
    run_all(projs, A_log, ds, h0=rand(B, ds, seed=3), reset=r)
    a = ops.gated_scan(projs, A_log, ds, reset=r)
    b = ops.gated_scan(projs, A_log, ds, reset=r.to(torch.uint8) * 255)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


@pytest.mark.parametrize("bad", [float("inf"), float("-inf"), float("nan")])
@pytest.mark.parametrize("at", [0, 100, 383, 384])
def test_reset_drops_infinities_and_nan(bad, at):
    """What a document holds does not reach the next one, nor its gradient the one before."""
    B, L, ds = 2, 600, 64
    projs, A_log = inputs(B, L, ds, F32)
    cut = 385
    r = torch.zeros(B, L, dtype=torch.bool, device=DEV)
    r[:, cut] = True
    dirty = projs.clone()
    dirty[:, at, ds:2 * ds] = bad
    h0 = torch.full((B, ds), bad, device=DEV)
    y, h, st = ops.gated_scan(dirty, A_log, ds, h0=h0, reset=r, return_states=True)
    ref = scan_ref(projs[:, cut:], A_log, ds, None, None, rand(B, L - cut, ds, seed=7))
    check(y[:, cut:], ref["y"], "y")
    check(h, ref["h_last"], "h_last")
    dy = torch.cat([torch.full((B, cut, ds), bad, device=DEV), rand(B, L - cut, ds, seed=7)], 1)
    dp, _, _ = ops.gated_scan_bwd(dy, dirty, A_log, st, ds, reset=r)
    check(dp[:, cut:], ref["dprojs"], "dprojs")
    # the other way: a gradient that is not finite after the cut stays there
    dy2 = torch.cat([rand(B, cut, ds, seed=9), torch.full((B, L - cut, ds), bad, device=DEV)], 1)
    st2 = ops.gated_scan(projs, A_log, ds, reset=r, return_states=True)[2]
    dp2, _, dh0 = ops.gated_scan_bwd(dy2, projs, A_log, st2, ds, reset=r, need_dh0=True)
    ref2 = scan_ref(projs[:, :cut], A_log, ds, None, None, rand(B, cut, ds, seed=9))
    check(dp2[:, :cut], ref2["dprojs"], "dprojs before the cut")
    check(dh0, ref2["dh0"], "dh0")


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_nan_stays_in_its_sequence_and_channel(dtype):
    B, L, ds = 3, 400, 72
    projs, A_log = inputs(B, L, ds, dtype)
    dirty = projs.clone()
    dirty[1, 150, ds + 5] = float("nan")
    y0, h0 = ops.gated_scan(projs, A_log, ds)
    y, h = ops.gated_scan(dirty, A_log, ds)
    assert bool(y[1, 150:, 5].isnan().all()) and bool(h[1, 5].isnan())
    y[1, 150:, 5] = y0[1, 150:, 5]
    h[1, 5] = h0[1, 5]
    assert torch.equal(y, y0) and torch.equal(h, h0)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("centre", [-30.0, -8.0, 0.0, 8.0, 25.0, 90.0])
def test_gate_range(dtype, centre):
    """Gates from nearly closed (softplus of -30) to decays that underflow at once."""
    B, L, ds = 2, 300, 64
    projs, A_log = inputs(B, L, ds, dtype)
    projs = projs.clone()
    projs[..., :ds] = (centre + 0.5 * rand(B, L, ds, seed=11)).to(dtype)
    run_all(projs, A_log, ds, h0=rand(B, ds, seed=3))


def test_gate_infinities():
    """dt = -inf keeps the state as it is; dt large forgets it."""
    projs, A_log = inputs(1, 200, 32, F32)
    projs = projs.clone()
    projs[:, 50:, :32] = float("-inf")
    y, h = ops.gated_scan(projs, A_log, 32)
    ref = scan_ref(projs, A_log, 32)
    assert torch.equal(ref["y"][0][:, 49], ref["h_last"][0])
    check(y, ref["y"], "y")
    check(h, ref["h_last"], "h_last")
    projs[:, 120, :32] = 1e4
    y, _ = ops.gated_scan(projs, A_log, 32)
    want = projs[:, 120, :32] * projs[:, 120, 64:] * projs[:, 120, 32:64]
    torch.testing.assert_close(y[:, 120], want, rtol=1e-6, atol=0)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_empty(dtype):
    projs, A_log = inputs(2, 0, 48, dtype)
    h0 = rand(2, 48, seed=3)
    y, h, st = ops.gated_scan(projs, A_log, 48, h0=h0, return_states=True)
    assert y.shape == (2, 0, 48) and torch.equal(h, h0)
    assert torch.equal(ops.gated_scan(projs, A_log, 48)[1], torch.zeros(2, 48, device=DEV))
    dh = rand(2, 48, seed=4)
    dp, dA, dh0 = ops.gated_scan_bwd(y, projs, A_log, st, 48, dh_last=dh, need_dh0=True)
    assert dp.shape == (2, 0, 144) and torch.equal(dh0, dh) and bool((dA == 0).all())
    none, A_log = inputs(0, 5, 48, dtype)
    y, h, st = ops.gated_scan(none, A_log, 48, return_states=True)
    assert y.shape == (0, 5, 48) and h.shape == (0, 48)
    assert bool((ops.gated_scan_bwd(y, none, A_log, st, 48)[1] == 0).all())


def test_windows_join():
    """A sequence run in windows with the state carried gives the whole sequence's outputs and,
    with the gradient carried back, its gradient."""
    B, L, ds, cut = 2, 700, 64, 333
    projs, A_log = inputs(B, L, ds, F32)
    dy, dh = rand(B, L, ds, seed=7), rand(B, ds, seed=8)
    ref = scan_ref(projs, A_log, ds, None, None, dy, dh)
    y1, h1, s1 = ops.gated_scan(projs[:, :cut], A_log, ds, return_states=True)
    y2, h2, s2 = ops.gated_scan(projs[:, cut:], A_log, ds, h0=h1, return_states=True)
    check(torch.cat([y1, y2], 1), ref["y"], "y")
    check(h2, ref["h_last"], "h_last")
    d2, A2, c = ops.gated_scan_bwd(dy[:, cut:], projs[:, cut:], A_log, s2, ds, dh_last=dh, need_dh0=True)
    d1, A1, _ = ops.gated_scan_bwd(dy[:, :cut], projs[:, :cut], A_log, s1, ds, dh_last=c)
    check(torch.cat([d1, d2], 1), ref["dprojs"], "dprojs")
    check(A1 + A2, ref["dA_log"], "dA_log")


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("B,ds", [(1, 1), (1, 768), (3, 65), (33, 256), (2, 1000)])
def test_step(dtype, B, ds):
    """Steps one by one give the scan's outputs and state (same arithmetic per step)."""
    T = 9
    projs, A_log = inputs(B, T, ds, dtype)
    reset = torch.zeros(B, T, dtype=torch.bool, device=DEV)
    reset[0, 4] = True
    h = rand(B, ds, seed=3)
    ref = scan_ref(projs, A_log, ds, h, reset)
    h0 = h.clone()
    ys = []
    for t in range(T):
        y, h2 = ops.gated_step(projs[:, t], A_log, h, ds, reset=reset[:, t])
        assert h2.data_ptr() == h.data_ptr()
        ys.append(y)
    check(torch.stack(ys, 1), ref["y"], "y")
    check(h, ref["h_last"], "h")
    h_out = torch.empty_like(h0)
    keep = h0.clone()
    buf = torch.full((B, ds + 3), 7.0, device=DEV, dtype=dtype)
    y, h2 = ops.gated_step(projs[:, 0], A_log, h0, ds, out=buf[:, 1:ds + 1], h_out=h_out)
    assert torch.equal(h0, keep) and h2.data_ptr() == h_out.data_ptr() and torch.equal(y, ys[0])
    assert bool((buf[:, 0] == 7.0).all()) and bool((buf[:, ds + 1:] == 7.0).all())


@pytest.mark.parametrize("a_dtype", [BF16, F32])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_A_log_type(dtype, a_dtype):
    projs, A_log = inputs(2, 300, 64, dtype)
    got = run_all(projs, A_log.to(a_dtype), 64)
    assert got["dA_log"].dtype == a_dtype


def test_repeats_bit_for_bit():
    projs, A_log = inputs(4, 3000, 200, BF16)
    dy = rand(4, 3000, 200, seed=7, dtype=BF16)
    first = None
    for _ in range(4):
        y, h, st = ops.gated_scan(projs, A_log, 200, return_states=True)
        dp, dA, dh0 = ops.gated_scan_bwd(dy, projs, A_log, st, 200, need_dh0=True)
        now = (y, h, st, dp, dA, dh0)
        if first is not None:
            assert all(torch.equal(a, b) for a, b in zip(first, now))
        first = now


def test_batch_rows_do_not_depend_on_each_other():
    projs, A_log = inputs(3, 500, 96, BF16)
    y, h = ops.gated_scan(projs, A_log, 96)
    y1, h1 = ops.gated_scan(projs[1:2], A_log, 96)
    torch.testing.assert_close(y[1:2].float(), y1.float(), rtol=2 ** -7, atol=1e-6)
    torch.testing.assert_close(h[1:2], h1, rtol=1e-5, atol=1e-6)


def test_other_stream_and_graph():
    projs, A_log = inputs(2, 900, 128, BF16)
    want = ops.gated_scan(projs, A_log, 128)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = ops.gated_scan(projs, A_log, 128)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    dy = rand(2, 900, 128, seed=7, dtype=BF16)
    st = ops.gated_scan(projs, A_log, 128, return_states=True)[2]
    grad = ops.gated_scan_bwd(dy, projs, A_log, st, 128)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y, h, st2 = ops.gated_scan(projs, A_log, 128, return_states=True)
        dp, dA, _ = ops.gated_scan_bwd(dy, projs, A_log, st2, 128)
    for _ in range(3):
        y.zero_(), dp.zero_()
        graph.replay()
        assert torch.equal(y, want[0]) and torch.equal(dp, grad[0]) and torch.equal(dA, grad[1])
    assert _lib.load().hdc_device_error(1) == 0


def test_offsets_beyond_32_bits():
    """projs and dprojs of more than 2^31 elements; the last rows are a document of their own."""
    ds, B = 512, 1
    L = 2 ** 31 // (3 * ds) + 300
    projs = torch.empty(B, L, 3 * ds, device=DEV, dtype=BF16)
    projs.normal_(generator=torch.Generator(device=DEV).manual_seed(1))
    A_log = torch.zeros(ds, device=DEV)
    reset = torch.zeros(B, L, dtype=torch.bool, device=DEV)
    cut = L - 200
    reset[:, cut] = True
    y, h, st = ops.gated_scan(projs, A_log, ds, reset=reset, return_states=True)
    dy = torch.zeros(B, L, ds, device=DEV, dtype=BF16)
    dy[:, cut:] = rand(B, L - cut, ds, seed=7, dtype=BF16)
    dp, _, _ = ops.gated_scan_bwd(dy, projs, A_log, st, ds, reset=reset)
    ref = scan_ref(projs[:, cut:], A_log, ds, None, None, dy[:, cut:])
    check(y[:, cut:], ref["y"], "y")
    check(h, ref["h_last"], "h_last")
    check(dp[:, cut:], ref["dprojs"], "dprojs")
    assert bool((dp[:, cut - 1000:cut] == 0).all())


# ------------------------------------------------------------------ autograd
def test_gradient_against_differences():
    """Directional derivatives of the definition, by central differences in 64 bits (step 1e-6:
    truncation 1e-12, rounding 1e-10 of the terms' size; the fp32 gradient's own rounding, 1e-5
    of their size, decides)."""
    B, L, ds = 2, 150, 20
    projs, A_log = inputs(B, L, ds, F32)
    h0 = rand(B, ds, seed=3)
    reset = torch.rand(B, L, generator=torch.Generator(device=DEV).manual_seed(5), device=DEV) < 0.02
    dy, dh = rand(B, L, ds, seed=7), rand(B, ds, seed=8)
    leaves = [t.clone().requires_grad_() for t in (projs, A_log, h0)]
    y, h = recurrent.gated_scan(leaves[0], leaves[1], ds, h0=leaves[2], reset=reset)
    grads = torch.autograd.grad([y, h], leaves, [dy, dh])

    def loss(p, a, s):
        v = scan_values(p, a, ds, s, reset)
        return float((v * dy.double()).sum() + (v[:, -1] * dh.double()).sum())

    base = [t.double() for t in (projs, A_log, h0)]
    for i, gr in enumerate(grads):
        for seed in range(3):
            v = rand(*gr.shape, seed=100 + seed).double()
            up, down = list(base), list(base)
            up[i], down[i] = base[i] + 1e-6 * v, base[i] - 1e-6 * v
            want = (loss(*up) - loss(*down)) / 2e-6
            size = float((gr.double() * v).abs().sum())
            assert abs(float((gr.double() * v).sum()) - want) <= 1e-5 * size + 1e-6 * abs(loss(*base)), (i, seed)


def test_autograd_inputs():
    """Only what is asked for is returned; extra columns get zero; y or h_last alone works."""
    B, L, ds = 2, 130, 16
    projs, A_log = inputs(B, L, ds, F32, extra=7)
    p = projs.clone().requires_grad_()
    y, h = recurrent.gated_scan(p, A_log, ds)
    gy, = torch.autograd.grad(y.sum(), p)
    assert gy.shape == p.shape and bool((gy[..., 3 * ds:] == 0).all())
    ref = scan_ref(projs, A_log, ds, None, None, torch.ones(B, L, ds, device=DEV))
    check(gy[..., :3 * ds], ref["dprojs"], "dprojs")
    y, h = recurrent.gated_scan(p, A_log, ds)
    gh, = torch.autograd.grad(h.sum(), p)
    ref = scan_ref(projs, A_log, ds, None, None, torch.zeros(B, L, ds, device=DEV), torch.ones(B, ds, device=DEV))
    check(gh[..., :3 * ds], ref["dprojs"], "dprojs of h_last")
    a = A_log.clone().requires_grad_()
    s = rand(B, ds, seed=3).requires_grad_()
    y, h = recurrent.gated_scan(projs, a, ds, h0=s)
    ga, gs = torch.autograd.grad(y.square().sum(), (a, s))
    assert ga.shape == a.shape and gs.shape == s.shape
    with torch.no_grad():
        assert recurrent.gated_scan(p, a, ds)[0].grad_fn is None


def test_second_order_raises():
    projs, A_log = inputs(1, 20, 16, F32)
    p = projs.clone().requires_grad_()
    y, _ = recurrent.gated_scan(p, A_log, 16)
    with pytest.raises(RuntimeError, match="once"):
        torch.autograd.grad(y.sum(), p, create_graph=True)
    z = recurrent.group_norm_act(p, 3, act="silu")
    with pytest.raises(RuntimeError, match="once"):
        torch.autograd.grad(z.sum(), p, create_graph=True)


# ------------------------------------------------------------------ refusals
def test_refusals():
    projs, A_log = inputs(2, 10, 16, F32)
    with pytest.raises(ValueError, match="3\\*d_state"):
        ops.gated_scan(projs, torch.zeros(17, device=DEV), 17)
    with pytest.raises(ValueError, match="A_log"):
        ops.gated_scan(projs, torch.zeros(15, device=DEV), 16)
    with pytest.raises(ValueError, match="column stride"):
        ops.gated_scan(projs.transpose(1, 2).contiguous().transpose(1, 2), A_log, 16)
    with pytest.raises(ValueError, match="h0"):
        ops.gated_scan(projs, A_log, 16, h0=torch.zeros(2, 15, device=DEV))
    with pytest.raises(ValueError, match="reset"):
        ops.gated_scan(projs, A_log, 16, reset=torch.zeros(2, 9, dtype=torch.bool, device=DEV))
    with pytest.raises(ValueError, match="reset"):
        ops.gated_scan(projs, A_log, 16, reset=torch.zeros(2, 10, device=DEV))
    with pytest.raises(TypeError, match="dtype"):
        ops.gated_scan(projs.half(), A_log, 16)
    with pytest.raises(TypeError, match="dtype"):
        ops.gated_scan(projs, A_log.double(), 16)
    with pytest.raises(ValueError, match="out"):
        ops.gated_scan(projs, A_log, 16, out=torch.empty(2, 10, 15, device=DEV))
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.gated_scan(projs.cpu(), A_log, 16)
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.gated_scan(projs, A_log, 16, reset=torch.zeros(2, 10, dtype=torch.bool))
    st = ops.gated_scan(projs, A_log, 16, return_states=True)[2]
    dy = torch.zeros(2, 10, 16, device=DEV)
    with pytest.raises(ValueError, match="states"):
        ops.gated_scan_bwd(dy, projs, A_log, st.repeat(1, 2, 1), 16)
    with pytest.raises(ValueError, match="dy"):
        ops.gated_scan_bwd(dy[:, :9], projs, A_log, st, 16)
    with pytest.raises(TypeError, match="mismatch"):
        ops.gated_scan_bwd(dy.bfloat16(), projs, A_log, st, 16)
    with pytest.raises(ValueError, match="dh_last"):
        ops.gated_scan_bwd(dy, projs, A_log, st, 16, dh_last=torch.zeros(1, 16, device=DEV))
    with pytest.raises(ValueError, match="h must"):
        ops.gated_step(projs[:, 0], A_log, torch.zeros(2, 16, device=DEV, dtype=torch.bfloat16), 16)
    with pytest.raises(ValueError, match="reset"):
        ops.gated_step(projs[:, 0], A_log, torch.zeros(2, 16, device=DEV), 16,
                       reset=torch.zeros(3, dtype=torch.bool, device=DEV))
