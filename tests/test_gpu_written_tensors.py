"""Tensors that a call writes are known to autograd as written: what was saved of them before is not taken for what it was."""
import pytest
import torch

from hdcmamba_b200 import ops, training

pytestmark = pytest.mark.gpu


def test_versions():
    q, g = torch.randn(2, 3, 8, device="cuda"), torch.tensor([-0.1, -0.2, -1.0], device="cuda")
    s, s2, o = torch.zeros(2, 3, 8, 8, device="cuda"), torch.zeros(2, 3, 8, 8, device="cuda"), torch.empty_like(q)
    ids, w, y = torch.tensor([1, 2], device="cuda"), torch.randn(4, 8, device="cuda"), torch.empty(2, 8, device="cuda")
    d, x, p = torch.empty(4, 8, device="cuda"), torch.ones(50, device="cuda"), torch.nn.Parameter(torch.ones(5, device="cuda"))
    z, long = torch.empty(50, device="cuda"), torch.empty(2, 1, 3, 8, device="cuda")
    p.grad = torch.ones(5, device="cuda")
    calls = [
        (lambda: ops.decay_attention_step(q, q, q, g, s), [s], [q, g]),
        (lambda: ops.decay_attention_step(q, q, q, g, s, out=o, state_out=s2), [o, s2], [q, g, s]),
        (lambda: ops.decay_attention(q[:, None], q[:, None], q[:, None], g, out=long), [long], [q, g]),
        (lambda: ops.embedding(ids, w, out=y), [y], [ids, w]),
        (lambda: ops.embedding_bwd(y, ids, 4, out=d), [d], [y, ids]),
        (lambda: ops.clip_grads([x], 1.0), [x], []),
        (lambda: ops.clip_grads([x], 1.0, out=[z]), [z], [x]),
        (lambda: ops.clip_grads([x], None), [], [x]),
        (lambda: training.clip_grad_norm_([p], 1.0), [p.grad], [p]),
    ]
    for i, (call, written, read) in enumerate(calls):
        before = [t._version for t in written + read]
        call()
        after = [t._version for t in written + read]
        assert [a > b for a, b in zip(after, before)] == [True] * len(written) + [False] * len(read), i


def test_a_state_that_was_saved():
    q, g = torch.randn(1, 2, 8, device="cuda"), torch.tensor([-0.1, -0.2], device="cuda")
    s = torch.randn(1, 2, 8, 8, device="cuda")
    w = torch.ones_like(s).requires_grad_()
    loss = (w * s).sum()
    ops.decay_attention_step(q, q, q, g, s)
    with pytest.raises(RuntimeError, match="inplace"):
        loss.backward()


def test_inference_tensors():
    """They have no versions, and are written all the same."""
    with torch.inference_mode():
        q, g = torch.randn(1, 2, 8, device="cuda"), torch.tensor([-0.1, -0.2], device="cuda")
        s, x = torch.zeros(1, 2, 8, 8, device="cuda"), torch.ones(50, device="cuda")
        ops.decay_attention_step(q, q, q, g, s)
        ops.clip_grads([x], 1.0)
        assert torch.allclose(s, q[..., :, None] * q[..., None, :]) and (x < 1).all()
