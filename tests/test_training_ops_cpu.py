"""Arguments that decayed attention, the embedding and clipping refuse; sizes that the library computes.  Nothing here
launches a kernel: every call ends at a check."""
import ctypes

import pytest
import torch

from attn_ref import gradient, recur
from hdcmamba_b200 import _lib, ops, recurrent, training


def test_cpu_tensors_raise():
    q = torch.zeros(1, 2, 3, 8)
    g = torch.zeros(3)
    with pytest.raises(RuntimeError):
        ops.decay_attention(q, q, q, g)
    with pytest.raises(RuntimeError):
        recurrent.decay_attention(q, q, q, g)
    with pytest.raises(RuntimeError):
        ops.decay_attention_step(q[:, 0], q[:, 0], q[:, 0], g, torch.zeros(1, 3, 8, 8))
    with pytest.raises(RuntimeError):
        training.embedding(torch.zeros(3, dtype=torch.int64), torch.zeros(4, 8))
    with pytest.raises(RuntimeError):
        ops.embedding_bwd(torch.zeros(3, 8), torch.zeros(3, dtype=torch.int64), 4)
    with pytest.raises(RuntimeError):
        ops.clip_grads([torch.zeros(3)], 1.0)
    with pytest.raises(ValueError):
        ops.clip_grads([], 1.0)


# CPU tensors: sizes and types are looked at before the device, so a call that they allow ends there (RuntimeError)


def test_attention_refusals():
    q, g, s = torch.zeros(2, 5, 3, 8), torch.zeros(3), torch.zeros(2, 3, 8, 8)
    bad = [
        dict(q=q.half(), k=q.half(), v=q.half()), dict(k=q.bfloat16()), dict(k=torch.zeros(2, 4, 3, 8)),
        dict(v=torch.zeros(2, 5, 3, 9)), dict(log_decay=torch.zeros(4)), dict(log_decay=torch.zeros(2, 5, 3)),
        dict(state=torch.zeros(2, 3, 8, 9)), dict(state=s.bfloat16()), dict(state=s.transpose(2, 3)),
        dict(q=q[0], k=q[0], v=q[0]), dict(q=torch.zeros(2, 5, 8, 3).transpose(2, 3)),
        dict(out=torch.zeros(2, 5, 3, 7)), dict(out=q.bfloat16()), dict(out=torch.zeros(2, 5, 8, 3).transpose(2, 3)),
        dict(q=torch.zeros(1, 1, 1, 129), k=torch.zeros(1, 1, 1, 129), v=torch.zeros(1, 1, 1, 129), log_decay=torch.zeros(1)),
        dict(q=torch.zeros(1, 1, 0, 8), k=torch.zeros(1, 1, 0, 8), v=torch.zeros(1, 1, 0, 8), log_decay=torch.zeros(0)),
    ]
    for kw in bad:
        with pytest.raises((ValueError, TypeError)):
            ops.decay_attention(**(dict(q=q, k=q, v=q, log_decay=g) | kw))
    n = ops._size("hdc_decay_attn_state_slots", 0, 2, 5, 3, 8)
    st = torch.zeros(2, 3, n, 8, 8)
    for kw in (dict(do=q.bfloat16()), dict(do=q[:, :4]), dict(states=st[:, :2]), dict(states=st.double()),
               dict(dstate=s[:1])):
        with pytest.raises((ValueError, TypeError)):
            ops.decay_attention_bwd(**(dict(do=q, q=q, k=q, v=q, log_decay=g, states=st) | kw))
    r = torch.zeros(2, 3, 8)
    for kw in (dict(q=q), dict(state=s[:1]), dict(state_out=s.double()), dict(out=r[:1]), dict(k=r.bfloat16())):
        with pytest.raises((ValueError, TypeError)):
            ops.decay_attention_step(**(dict(q=r, k=r, v=r, log_decay=g, state=s) | kw))


def test_embedding_refusals():
    ids, w = torch.zeros(4, dtype=torch.int64), torch.zeros(10, 8)
    for kw in (dict(ids=ids.float()), dict(ids=ids.short()), dict(weight=w.half()), dict(weight=w.t()), dict(weight=w[0]),
               dict(weight=w[:, :0]), dict(out=torch.zeros(4, 9)), dict(out=torch.zeros(4, 8).bfloat16()),
               dict(out=torch.zeros(8, 4).t())):
        with pytest.raises((ValueError, TypeError)):
            ops.embedding(**(dict(ids=ids, weight=w) | kw))
    dy = torch.zeros(4, 8)
    for kw in (dict(dy=dy[:3]), dict(dy=dy.half()), dict(out=torch.zeros(9, 8)), dict(out=torch.zeros(8, 10).t()), dict(rows=0),
               dict(out=torch.zeros(10, 8).bfloat16())):
        with pytest.raises((ValueError, TypeError)):
            ops.embedding_bwd(**(dict(dy=dy, ids=ids, rows=10) | kw))


def test_clip_refusals():
    x = torch.zeros(4, 5)
    for grads, out in (([x.t()], None), ([x.half()], None), ([x], [x.bfloat16()]), ([x], [torch.zeros(21)]), ([x], []),
                       ([x], [torch.zeros(5, 4).t()]), ([x, x.long()], None)):
        with pytest.raises((ValueError, TypeError)):
            ops.clip_grads(grads, 1.0, out=out)


A = 0x10000  # an address that no call reads


def rc(name, *args):
    code = getattr(_lib.load(), name)(*args)
    return code, _lib.load().hdc_error_string().decode()


def attn_fwd(**kw):
    v = dict(dtype=1, q=A, k=A, v=A, st=(64, 32, 8), g=A, s0=None, o=A, ost=(64, 32, 8), s1=None, states=A, B=2, L=2, H=4, D=8) | kw
    return rc("hdc_decay_attn_fwd", v["dtype"], v["q"], *v["st"], v["k"], *v["st"], v["v"], *v["st"], v["g"], v["s0"], 1.0, v["o"],
              *v["ost"], v["s1"], v["states"], v["B"], v["L"], v["H"], v["D"], None)[0]


def test_checks_beside_the_operators(monkeypatch):
    monkeypatch.setattr(recurrent, "_require_cuda", lambda *t: None)
    monkeypatch.setattr(training, "_require_cuda", lambda *t: None)
    q, g = torch.zeros(2, 5, 3, 8), torch.zeros(3)
    with pytest.raises(ValueError, match="log_decay"):
        recurrent.decay_attention(q, q, q, g.requires_grad_())
    for bad in (-1, 10):
        with pytest.raises(ValueError, match="padding_idx"):
            training.embedding(torch.zeros(4, dtype=torch.int64), torch.zeros(10, 8), padding_idx=bad)
    for bad in (None, 3, "q"):
        with pytest.raises(TypeError):
            ops.decay_attention(bad, q, q, g)
        with pytest.raises(TypeError):
            ops.clip_grads([q, bad], 1.0)
    with pytest.raises(TypeError):
        ops.decay_attention(q, q, q, g, scale="1")
    with pytest.raises(TypeError):
        ops.clip_grads(5, 1.0)


def test_c_checks_attention():
    assert attn_fwd(dtype=2) == -1
    assert attn_fwd(D=129) == -2 and attn_fwd(D=0) == -2 and attn_fwd(H=0) == -2 and attn_fwd(L=-1) == -2 and attn_fwd(B=-1) == -2
    assert attn_fwd(L=2 ** 30 + 1) == -2 and attn_fwd(B=2 ** 30, H=4) == -2
    assert attn_fwd(q=None) == -4 and attn_fwd(L=4096, st=(1 << 20, 32, 8), ost=(1 << 20, 32, 8), states=None) == -4 and attn_fwd(g=None) == -4 and attn_fwd(o=None) == -4
    assert attn_fwd(q=A + 1) == -3 and attn_fwd(states=A + 2) == -3 and attn_fwd(dtype=0, o=A + 2) == -3
    # rows of o that overlap: each of the three strides too short
    for ost in ((64, 32, 7), (64, 31, 8), (63, 32, 8), (0, 32, 8), (64, 0, 8), (8, 8, 8)):
        assert attn_fwd(ost=ost) == -2, ost
    assert attn_fwd(B=0) == 0
    st = (64, 32, 8)

    def bwd(**kw):
        v = dict(dtype=1, dq=A, dk=A, dv=A, dst=st, ws=A, n=1 << 20, B=2, L=2, H=4, D=8, states=A) | kw
        return rc("hdc_decay_attn_bwd", v["dtype"], A, *st, A, *st, A, *st, A, *st, A, v["states"], None, 1.0, v["dq"], *v["dst"],
                  v["dk"], *v["dst"], v["dv"], *v["dst"], None, v["ws"], v["n"], v["B"], v["L"], v["H"], v["D"], None)[0]

    assert _lib.load().hdc_decay_attn_bwd_workspace_bytes(1, 2, 2, 4, 8) == 0  # one segment
    need = _lib.load().hdc_decay_attn_bwd_workspace_bytes(1, 2, 4096, 4, 8)
    assert need == 2 * 4 * 64 * 4 * _lib.load().hdc_decay_attn_state_slots(1, 2, 4096, 4, 8) > 0
    long = dict(L=4096, dst=(1 << 20, 32, 8))
    assert bwd(n=need - 1, **long) == -5 and bwd(ws=None, **long) == -5 and bwd(ws=A + 8, **long) == -3
    assert bwd(dq=None) == -4 and bwd(states=None) == -4
    assert bwd(dst=(64, 32, 4)) == -2 and bwd(dtype=7) == -1 and bwd(B=0) == 0

    def step(**kw):
        v = dict(dtype=1, q=A, s=A, o=A, ost=(32, 8), out=A, B=2, H=4, D=8) | kw
        return rc("hdc_decay_attn_step", v["dtype"], v["q"], 32, 8, A, 32, 8, A, 32, 8, A, v["s"], 1.0, v["o"], *v["ost"], v["out"],
                  v["B"], v["H"], v["D"], None)[0]

    assert step(dtype=3) == -1 and step(D=200) == -2 and step(q=None) == -4 and step(s=A + 1) == -3 and step(out=None) == -4
    assert step(ost=(32, 4)) == -2 and step(ost=(0, 8)) == -2 and step(B=0) == 0


def test_state_slots_are_a_function_of_the_sizes():
    n = _lib.load().hdc_decay_attn_state_slots
    for dtype in (0, 1):
        for B, L, H in ((1, 1, 1), (1, 64, 1), (1, 65, 1), (1, 32768, 12), (8, 4096, 16), (1000, 1000, 16), (1, 1 << 30, 1)):
            for D in (1, 64, 128):
                s = n(dtype, B, L, H, D)
                assert 1 <= s <= -(-L // 64) + 1 and B * H * s <= max(2 * B * H, 2048), (B, L, H, D, s)
        assert n(dtype, 1, 0, 1, 64) == 0 and n(dtype, 0, 5, 1, 64) == 0


def test_c_checks_embedding():
    def fwd(**kw):
        v = dict(dtype=1, ids=A, ib=8, t=A, ts=8, y=A, ys=8, N=4, rows=10, D=8) | kw
        return rc("hdc_embedding_fwd", v["dtype"], v["ids"], v["ib"], v["t"], v["ts"], v["y"], v["ys"], 1.0, v["N"], v["rows"], v["D"],
                  None)[0]

    assert fwd(dtype=2) == -1 and fwd(ib=2) == -1 and fwd(N=-1) == -2 and fwd(rows=0) == -2 and fwd(D=0) == -2 and fwd(D=65537) == -2
    assert fwd(ids=None) == -4 and fwd(t=A + 1) == -3 and fwd(ids=A + 4) == -3 and fwd(ys=7) == -2 and fwd(N=0) == 0

    def bwd(**kw):
        v = dict(dtype=0, ids=A, ib=8, dy=A, d=A, ds=8, ws=A, n=1 << 30, N=4, rows=10, D=8) | kw
        return rc("hdc_embedding_bwd", v["dtype"], v["ids"], v["ib"], v["dy"], 8, v["d"], v["ds"], 1.0, -1, v["ws"], v["n"], v["N"],
                  v["rows"], v["D"], None)[0]

    need = _lib.load().hdc_embedding_bwd_workspace_bytes(4, 10, 8)
    assert bwd(dtype=2) == -1 and bwd(ib=1) == -1 and bwd(n=need - 1) == -5 and bwd(ws=None) == -5 and bwd(ws=A + 4) == -3
    assert bwd(d=None) == -4 and bwd(dy=None) == -4 and bwd(dy=A + 2) == -3 and bwd(ds=4) == -2 and bwd(rows=2 ** 30 + 1) == -2


def test_c_checks_clip():
    def clip(sizes=(4, 4), grads=(A, A + 64), outs=(A, A + 64), types=(0, 0), max_norm=1.0, norm=A, ws=A, n=None, bytes_=1 << 20):
        m = len(sizes)
        P = ctypes.c_void_p * m
        return rc("hdc_clip_grads", m if n is None else n, (ctypes.c_int * m)(*types), P(*grads), P(*outs) if outs else None,
                  (ctypes.c_int64 * m)(*sizes), max_norm, norm, ws, bytes_, None)

    assert clip(types=(0, 5))[0] == -1 and clip(sizes=(4, -1))[0] == -2 and clip(n=-1)[0] == -2
    assert clip(grads=(A, None))[0] == -4 and clip(norm=None)[0] == -4 and clip(ws=None)[0] == -4
    assert clip(bytes_=100)[0] == -5 and clip(ws=A + 8)[0] == -3 and clip(norm=A + 2)[0] == -3 and clip(grads=(A, A + 65))[0] == -3
    assert clip(max_norm=-1.0)[0] == -2 and clip(max_norm=float("nan"))[0] == -2
    # the same tensor twice, outputs that overlap one another or another's gradient
    assert clip(grads=(A, A), outs=(A, A))[0] == -2
    assert clip(outs=(A, A + 8))[0] == -2 and clip(outs=(A + 128, A + 132))[0] == -2
    assert clip(outs=(A + 4, A + 64))[0] == -2 and clip(outs=(A + 64, A + 512))[0] == -2


def test_definition_against_autograd_and_differences():
    """The reverse recurrence of the tests is the derivative of the recurrence."""
    gen = torch.Generator().manual_seed(0)
    q, k, v, do = (torch.randn(2, 9, 2, 5, generator=gen, dtype=torch.float64) for _ in range(4))
    s, ds = (torch.randn(2, 2, 5, 5, generator=gen, dtype=torch.float64) for _ in range(2))
    g = torch.tensor([-0.1, -1.0], dtype=torch.float64)
    leaves = [x.requires_grad_() for x in (q, k, v, s)]
    o, e = recur(q, k, v, g, 0.3, s)
    auto = torch.autograd.grad([o, e], leaves, [do, ds])
    with torch.no_grad():
        for a, b in zip(auto, gradient(q, k, v, g, 0.3, s, do, ds)):
            assert torch.allclose(a, b, rtol=1e-12, atol=1e-12)
    assert torch.autograd.gradcheck(lambda *x: recur(x[0], x[1], x[2], g, 0.3, x[3]), [x[:, :3].detach().requires_grad_() for x in (q, k, v)] + [s])
