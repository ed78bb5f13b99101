"""Infinities and NaN on the masked side of the diagonal: a token reaches no output before it, as in the recurrence (and
no gradient of a token behind it, through the state's gradient, which runs backwards).  What it does not reach is
compared with the definition in 64 bits (bounds: attn_ref.py)."""
import ctypes

import pytest
import torch

from attn_ref import close, gradient, recur
from hdcmamba_b200 import _lib, ops

pytestmark = pytest.mark.gpu
F32, BF16 = torch.float32, torch.bfloat16
# one segment and several, of 64 and of 128 tokens a chunk; every padded width
CASES = [(32, 100), (40, 64), (64, 40), (64, 300), (128, 200), (20, 257), (64, 2100), (40, 2500), (96, 700), (1, 130)]


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("bad", [float("inf"), float("-inf"), float("nan")])
@pytest.mark.parametrize("D,L", CASES)
def test_masked_tokens_that_are_not_finite(dtype, D, L, bad):
    bf16 = dtype == BF16
    g = torch.Generator().manual_seed(D + L)
    B, H = 2, 2
    q, k, v, do = (torch.randn(B, L, H, D, generator=g).to(dtype).cuda() for _ in range(4))
    ld = torch.tensor([-0.02, -0.4]).cuda()
    a = [x.double().cpu() for x in (q, k, v)]
    ld64, d64 = ld.double().cpu(), do.double().cpu()
    names = ("o", "dq", "dk", "dv")
    ref = [recur(*a, ld64, 0.3)[0], *gradient(*a, ld64, 0.3, None, d64, None)[:3]]
    a = [x.abs() for x in a]
    size = [recur(*a, ld64, 0.3)[0], *gradient(*a, ld64, 0.3, None, d64.abs(), None)[:3]]

    def clean(name, got, rows):
        """Rows `rows` of batch 0 and head 1, and every other batch and head, are what they are without the token."""
        i = names.index(name)
        for b in range(B):
            for h in range(H):
                r = rows if (b, h) == (0, 1) else slice(None)
                close(name, *(x[b:b + 1, r, h:h + 1] for x in (got, ref[i], size[i])), bf16)

    def spoiled(x, t):
        y = x.clone()
        y[0, t, 1, t % D] = bad
        return y

    st = ops.decay_attention(q, k, v, ld, 0.3, return_states=True)[2]
    for t in {L - 1, L // 2, 37 % L, 0}:
        near = slice(t, min(t + 8, L))  # (farther on infinity may meet a decay that has become zero)
        o, _ = ops.decay_attention(q, spoiled(k, t), v, ld, 0.3)
        clean("o", o, slice(0, t))
        assert not torch.isfinite(o[0, near, 1]).any()
        o, _ = ops.decay_attention(q, k, spoiled(v, t), ld, 0.3)
        clean("o", o, slice(0, t))
        assert not torch.isfinite(o[0, near, 1, t % D]).any()
        # the gradient of o_t: dq_t, and dk and dv of the tokens up to t
        _, dk, dv, _ = ops.decay_attention_bwd(spoiled(do, t), q, k, v, ld, st, 0.3)
        clean("dk", dk, slice(t + 1, L))
        clean("dv", dv, slice(t + 1, L))
        near = slice(max(t - 7, 0), t + 1)
        assert not torch.isfinite(dk[0, near, 1]).any() and not torch.isfinite(dv[0, near, 1, t % D]).any()
        # q_t likewise, and no dq
        dq, dk, dv, _ = ops.decay_attention_bwd(do, spoiled(q, t), k, v, ld, st, 0.3)
        clean("dq", dq, slice(None))
        clean("dk", dk, slice(t + 1, L))
        clean("dv", dv, slice(t + 1, L))
        # k_t and v_t: dq of the tokens from t on
        for x in ((q, spoiled(k, t), v), (q, k, spoiled(v, t))):
            clean("dq", ops.decay_attention_bwd(do, *x, ld, st, 0.3)[0], slice(0, t))


def forward(q, k, v, ld, state, state_out):
    """The C entry point: the state behind the sequence may take the place of the one before it."""
    B, L, H, D = q.shape
    dtype, o = (1 if q.dtype == BF16 else 0), torch.empty_like(q)
    n = ops._size("hdc_decay_attn_state_slots", dtype, B, L, H, D)
    states = torch.empty(B, H, n, D, D, device="cuda")
    st = q.stride()[:3]
    at = [ctypes.c_void_p(x.data_ptr()) for x in (q, k, v, ld, state, o, state_out, states)]
    _lib.call("hdc_decay_attn_fwd", dtype, at[0], *st, at[1], *st, at[2], *st, at[3], at[4], 0.3, at[5], *st, at[6], at[7], B, L, H, D,
              ctypes.c_void_p(torch.cuda.current_stream().cuda_stream))
    return o, state_out


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("D,L", [(32, 100), (64, 40), (128, 100), (64, 600), (64, 2100)])
@pytest.mark.parametrize("t", [None, 30])
def test_a_state_in_place(dtype, D, L, t):
    """With tokens that are all finite, and with one that is not."""
    g = torch.Generator().manual_seed(D + L)
    q, k, v = (torch.randn(2, L, 2, D, generator=g).to(dtype).cuda() for _ in range(3))
    ld, s = torch.tensor([-0.02, -0.4]).cuda(), torch.randn(2, 2, D, D, generator=g).cuda()
    if t is not None:
        v[0, t, 1, 3] = float("nan")
    want = forward(q, k, v, ld, s, torch.empty_like(s))
    got = forward(q, k, v, ld, s, s)
    for a, b in zip(got, want):
        assert torch.equal(a.nan_to_num(7.0), b.nan_to_num(7.0))
    assert torch.isfinite(want[0][0, :t]).all()


def test_products_of_outputs_that_overflow():
    """Finite outputs of 1e25: the check's products overflow, the outputs keep their bits."""
    g = torch.Generator().manual_seed(3)
    for dtype in (F32, BF16):
        for D, L in ((64, 300), (64, 2100), (128, 100), (32, 200)):
            q, k, v = (torch.randn(1, L, 2, D, generator=g).to(dtype).cuda() for _ in range(3))
            ld = torch.tensor([-0.02, -0.4]).cuda()
            o, e = ops.decay_attention(q, k, v, ld)
            big, e2 = ops.decay_attention(q, k, v * 2.0 ** 80, ld)
            assert torch.equal(big, o * 2.0 ** 80) and torch.equal(e2, e * 2.0 ** 80)
