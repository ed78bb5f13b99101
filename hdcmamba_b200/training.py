"""What a training step of an LM needs beside its layers (hdcmamba_b200/recurrent.py): the token
embedding with its gradient, and clipping by the norm over all gradients.

    h = embedding(ids, lm.embedding.weight)           # rows, differentiable
    loss.backward()
    norm = clip_grad_norm_(model.parameters(), 1.0)   # stays on the device
    optimizer.step()

There is no CPU path: CPU inputs raise.
"""
import torch

from . import _lib, ops
from .model import _require_cuda
from .recurrent import _no_tangents

__all__ = ["embedding", "clip_grad_norm_"]


def embedding(ids, weight, scale=1.0, padding_idx=None):
    """Differentiable ``ops.embedding`` (any number of times): ids.shape + [D].  ``padding_idx``: an id whose tokens take no
    part in the gradient (their rows are looked up like any other)."""
    _require_cuda(ids)
    _no_tangents(weight)
    if padding_idx is not None and not 0 <= padding_idx < weight.shape[0]:
        raise ValueError(f"padding_idx {padding_idx} is outside the table of {weight.shape[0]} rows")
    if torch.is_grad_enabled() and weight.requires_grad:
        return _lib.host().embedding_train(ids, weight, scale, padding_idx)  # a C++ autograd node
    return ops.embedding(ids, weight, scale)


@torch.no_grad()
def clip_grad_norm_(parameters, max_norm):
    """Scale the gradients of ``parameters`` (a tensor or an iterable) in place so that the norm over all
    of them is at most ``max_norm``; returns the norm before (fp32 on the device, which the host does
    not wait for).  Gradients are fp32 or bf16, mixed as they come; parameters without one are left out."""
    parameters = [parameters] if isinstance(parameters, torch.Tensor) else list(parameters)
    grads = [p.grad for p in parameters if p.grad is not None]
    if not grads:
        return torch.zeros((), device=parameters[0].device if parameters else None)
    if all(g.is_contiguous() for g in grads):
        return ops.clip_grads(grads, max_norm)
    # gradients in another order of memory: scaled in a copy
    rows = [g.contiguous() for g in grads]
    norm = ops.clip_grads(rows, max_norm)
    for g, r in zip(grads, rows):
        if r is not g:
            g.copy_(r)
    return norm
