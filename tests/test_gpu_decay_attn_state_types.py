"""A state of another type or order of memory: the call takes it with and without gradients alike."""
import pytest
import torch

from hdcmamba_b200 import recurrent

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("change", [lambda s: s.bfloat16(), lambda s: s.double(), lambda s: s.transpose(2, 3).contiguous().transpose(2, 3)])
def test_with_and_without_gradients(change):
    g = torch.Generator().manual_seed(1)
    q = torch.randn(2, 40, 2, 16, generator=g).cuda()
    ld, s = torch.tensor([-0.1, -1.0]).cuda(), change(torch.randn(2, 2, 16, 16, generator=g).cuda())
    want = recurrent.decay_attention(q.clone().requires_grad_(), q, q, ld, 0.5, s)
    with torch.no_grad():
        got = recurrent.decay_attention(q, q, q, ld, 0.5, s)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
