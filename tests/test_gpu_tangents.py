"""Forward-mode derivatives: the operators that have none refuse a tangent instead of dropping it."""
import pytest
import torch
import torch.autograd.forward_ad as fwd

from hdcmamba_b200 import recurrent, training

pytestmark = pytest.mark.gpu


def calls(dual):
    """Each operator's call with one input made dual."""
    r = lambda *s: torch.randn(*s, device="cuda")  # noqa: E731
    q, g, s = r(1, 5, 2, 8), -torch.rand(2, device="cuda"), r(1, 2, 8, 8)
    att = recurrent.decay_attention
    yield lambda: att(dual(q), q, q, g)
    yield lambda: att(q, dual(q), q, g)
    yield lambda: att(q, q, dual(q), g)
    yield lambda: att(q, q, q, dual(g))
    yield lambda: att(q, q, q, g, 1.0, dual(s))
    yield lambda: training.embedding(torch.tensor([1, 2], device="cuda"), dual(r(4, 8)))
    p, a, h = r(1, 5, 24), r(8), r(1, 8)
    yield lambda: recurrent.gated_scan(dual(p), a, 8)
    yield lambda: recurrent.gated_scan(p, dual(a), 8)
    yield lambda: recurrent.gated_scan(p, a, 8, h0=dual(h))
    x, w = r(4, 16), r(16)
    yield lambda: recurrent.group_norm_act(dual(x), 2, w, w)
    yield lambda: recurrent.group_norm_act(x, 2, dual(w), w)
    ln, conv = torch.nn.LayerNorm(8).cuda(), torch.nn.Conv1d(8, 8, 4, groups=8, padding=3).cuda()
    yield lambda: recurrent.norm_conv1d(dual(r(1, 5, 8)), ln, conv)


@pytest.mark.parametrize("grad", [False, True])
def test_a_tangent_is_refused(grad):
    with fwd.dual_level():
        n = 0
        for call in calls(lambda x: fwd.make_dual(x.requires_grad_(grad), torch.ones_like(x))):
            with pytest.raises((RuntimeError, ValueError)):
                call()
            n += 1
        assert n == 12
        for call in calls(lambda x: x):  # a level alone refuses nothing
            call()
