"""Infinities and NaN on the masked side of the diagonal: a token reaches no output before it, as in the recurrence (and
no gradient of a token behind it, through the state's gradient, which runs backwards).  What it does not reach is
compared with the definition in 64 bits (bounds: attn_ref.py)."""
import pytest
import torch

from attn_ref import close, gradient, recur
from hdcmamba_b200 import ops

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
