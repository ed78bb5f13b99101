"""Gradients scaled in place have the bits of gradients scaled into other buffers."""
import pytest
import torch

from hdcmamba_b200 import ops, training

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("lead", [0, 1, 5])
def test_in_place_and_elsewhere(dtype, lead):
    """Whole pieces and parts of one, at any distance from a 16-byte border, more pieces than CTAs."""
    g = torch.Generator(device="cuda").manual_seed(lead)
    sizes = [13, 8192, 30001, 1, 16384, 6_000_011, 4096]
    flat = torch.randn(lead + sum(sizes), generator=g, device="cuda").to(dtype)
    grads = list(flat[lead:].split(sizes))
    other = [torch.empty_like(x) for x in grads]
    n1 = ops.clip_grads(grads, 2.0, out=other)
    n2 = ops.clip_grads(grads, 2.0)
    assert torch.equal(n1, n2) and all(torch.equal(a, b) for a, b in zip(grads, other))


def test_the_norm_of_no_gradients_is_on_the_parameters_device():
    p = torch.nn.Parameter(torch.ones(3, device="cuda"))
    for params in (p, [p], iter([p])):
        norm = training.clip_grad_norm_(params, 1.0)
        assert norm.device == p.device and norm.dtype == torch.float32 and norm == 0
    assert training.clip_grad_norm_([], 1.0) == 0
