"""Tokens that are not finite, in heads narrower than the width that a kernel pads them to: the padding stays zero, so
an output that such a token makes infinite reaches no other chunk.  A row of x (q for o; do for dq, v for dk, k for dv)
enters its own output alone, whatever it holds: every other row has the bits that it has without it."""
import pytest
import torch

from hdcmamba_b200 import ops

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16


def inputs(D, L, seed):
    g = torch.Generator().manual_seed(seed)
    B, H = 2, 20
    q, k, v, do = (torch.randn(B, L, H, D, generator=g).to(BF16).cuda() for _ in range(4))
    return q, k, v, do, -torch.rand(H, generator=g).cuda()


def same_but_for(got, want, t):
    keep = torch.ones(want.shape[:3], dtype=torch.bool, device="cuda")
    keep[0, t, 0] = False
    return torch.equal(got[keep], want[keep])


@pytest.mark.parametrize("bad", [float("inf"), float("nan")])
@pytest.mark.parametrize("D,L", [(3, 256), (20, 256), (24, 500), (40, 256), (48, 500), (80, 256), (96, 256), (128, 256), (96, 1100)])
def test_a_row_of_x_reaches_its_own_output_alone(D, L, bad):
    q, k, v, do, ld = inputs(D, L, D)
    o, e, st = ops.decay_attention(q, k, v, ld, 0.3, return_states=True)
    dq, dk, dv, _ = ops.decay_attention_bwd(do, q, k, v, ld, st, 0.3)

    def spoiled(x, t):
        y = x.clone()
        y[0, t, 0, 0] = bad
        return y

    for t in (3, L - 2):
        got, after = ops.decay_attention(spoiled(q, t), k, v, ld, 0.3)
        assert same_but_for(got, o, t) and torch.equal(after, e)
        assert same_but_for(ops.decay_attention_bwd(spoiled(do, t), q, k, v, ld, st, 0.3)[0], dq, t)
        assert same_but_for(ops.decay_attention_bwd(do, q, k, spoiled(v, t), ld, st, 0.3)[1], dk, t)
        assert same_but_for(ops.decay_attention_bwd(do, q, spoiled(k, t), v, ld, st, 0.3)[2], dv, t)
