"""Outputs that lie in an input's memory are refused: other CTAs would still read it.  The check comes before the device's,
so CPU tensors show it; calls that are allowed end at the device's check."""
import pytest
import torch

from hdcmamba_b200 import _lib, ops


def refused(call):
    with pytest.raises(_lib.HdcError, match="overlap"):
        call()


def allowed(call):
    with pytest.raises(RuntimeError, match="CPU"):
        call()


def test_embedding():
    ids, flat = torch.zeros(4, dtype=torch.int64), torch.zeros(200)
    w = flat[:80].view(10, 8)
    refused(lambda: ops.embedding(ids, w, out=flat[:32].view(4, 8)))
    refused(lambda: ops.embedding(ids, w, out=flat[64:96].view(4, 8)))
    allowed(lambda: ops.embedding(ids, w, out=flat[80:112].view(4, 8)))
    words = torch.zeros(64)
    refused(lambda: ops.embedding(words.view(torch.int32)[:4], w, out=words[:32].view(4, 8)))
    dy = flat[:32].view(4, 8)
    refused(lambda: ops.embedding_bwd(dy, ids, 10, out=flat[24:104].view(10, 8)))
    allowed(lambda: ops.embedding_bwd(dy, ids, 10, out=flat[32:112].view(10, 8)))


def test_attention():
    flat, g = torch.zeros(2000), torch.zeros(3)
    q, k, v = (torch.zeros(2, 5, 3, 8) for _ in range(3))
    for x in (q, k, v):
        refused(lambda: ops.decay_attention(q, k, v, g, out=x))
    s = flat[:384].view(2, 3, 8, 8)
    refused(lambda: ops.decay_attention(q, k, v, g, state=s, out=flat[100:340].view(2, 5, 3, 8)))
    # slices of one projection beside each other
    p = torch.zeros(2, 5, 4 * 24)
    views = [t.unflatten(-1, (3, 8)) for t in p.split(24, -1)]
    allowed(lambda: ops.decay_attention(*views[:3], g, out=views[3]))
    refused(lambda: ops.decay_attention(*views[:3], g, out=views[2]))


def test_step():
    flat, g = torch.zeros(2000), torch.zeros(3)
    q, k, v = (torch.zeros(2, 3, 8) for _ in range(3))
    s, half = flat[:384].view(2, 3, 8, 8), flat[192:576].view(2, 3, 8, 8)
    allowed(lambda: ops.decay_attention_step(q, k, v, g, s))
    allowed(lambda: ops.decay_attention_step(q, k, v, g, s, state_out=s))
    allowed(lambda: ops.decay_attention_step(q, k, v, g, s, state_out=flat[384:768].view(2, 3, 8, 8)))
    refused(lambda: ops.decay_attention_step(q, k, v, g, s, state_out=half))
    refused(lambda: ops.decay_attention_step(q, k, v, g, s, out=flat[:48].view(2, 3, 8)))
    for x in (q, k, v):
        refused(lambda: ops.decay_attention_step(q, k, v, g, s, out=x))
    refused(lambda: ops.decay_attention_step(flat[:48].view(2, 3, 8), k, v, g, s))
