"""Gradients that nothing but the call holds: a generator's tensors live until the kernels have read them."""
import math

import pytest
import torch

from hdcmamba_b200 import ops

pytestmark = pytest.mark.gpu


def test_tensors_of_a_generator():
    """The norm of temporaries of many sizes, several of them as large as the norm's own and the call's workspace."""
    g = torch.Generator().manual_seed(1)
    sizes = [1, 100, 592, 1184, 1, 5000, 1, 9472 // 4, 70000] * 8
    xs = [torch.randn(n, generator=g).cuda().bfloat16() for n in sizes]
    want = math.sqrt(sum(float(x.double().square().sum()) for x in xs))
    for _ in range(3):
        got = ops.clip_grads((x.float() for x in xs), None)
        assert abs(float(got) - want) <= 20 * 2.0 ** -24 * want
    for many in (map(torch.Tensor.float, xs), (x.float() for x in xs)):
        assert torch.equal(ops.clip_grads(many, None), got)


def test_outputs_that_a_generator_makes():
    """Scaled into memory that only the call holds: nothing else is written."""
    xs = [torch.full((n,), 2.0, device="cuda") for n in (1, 100, 2368, 50000)]
    free = [torch.empty_like(x) for x in xs]
    del free
    norm = ops.clip_grads(xs, 1.0, out=(torch.empty_like(x) for x in xs))
    assert abs(float(norm) - 2 * math.sqrt(52469)) <= 20 * 2.0 ** -24 * float(norm) and all((x == 2).all() for x in xs)


def test_tensors_live_until_the_launch():
    """``max_norm`` is turned into a number last: then the generator's tensors are still there.  Nothing is launched."""
    class Number:
        def __float__(self):
            self.there = torch.cuda.memory_allocated() - before
            raise KeyError("seen")

    x, n = torch.ones(1 << 20, device="cuda"), Number()
    before = torch.cuda.memory_allocated()
    with pytest.raises(KeyError):
        ops.clip_grads((x * k for k in range(1, 5)), n)
    assert n.there >= 4 * (4 << 20)
