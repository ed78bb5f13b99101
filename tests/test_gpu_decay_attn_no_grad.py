"""Decays that are parameters: refused where their gradient would be missing, taken where none is wanted."""
import pytest
import torch

from hdcmamba_b200 import ops, recurrent

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("mode", [torch.no_grad, torch.inference_mode])
def test_decays_that_are_a_parameter(mode):
    q = torch.randn(1, 70, 2, 32, generator=torch.Generator().manual_seed(1)).cuda()
    ld = torch.nn.Parameter(torch.tensor([-0.1, -1.0], device="cuda"))
    want = ops.decay_attention(q, q, q, ld.detach())
    with mode():
        got = recurrent.decay_attention(q, q, q, ld)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    with pytest.raises(ValueError, match="log_decay"):
        recurrent.decay_attention(q, q, q, ld)
