"""A training step and generation of a small LM made of the operators: embedding, norm + conv, decayed attention,
group norm, tied head, clipping; the gradients against the same model in 64 bits on the CPU."""
import pytest
import torch
import torch.nn.functional as F

from attn_ref import recur
from hdcmamba_b200 import ops, recurrent, training
from hdcmamba_b200.lm import HdcMambaLM

pytestmark = pytest.mark.gpu
V, D, H, HD, L, B = 50, 32, 2, 16, 70, 2


class Layer(torch.nn.Module):
    def __init__(self):
        super().__init__()
        self.norm = torch.nn.LayerNorm(D)
        self.conv = torch.nn.Conv1d(D, D, kernel_size=4, groups=D, padding=3, bias=True)
        self.qkv = torch.nn.Linear(D, 3 * H * HD)
        self.group_norm = torch.nn.GroupNorm(H, H * HD)
        self.out = torch.nn.Linear(H * HD, D, bias=False)
        self.register_buffer("log_decay", -torch.tensor([0.02, 0.3]))


def model():
    torch.manual_seed(0)
    m = torch.nn.Module()
    m.embedding = torch.nn.Embedding(V, D)
    m.layer = Layer()
    return m


def heads(x):
    return [t.unflatten(-1, (H, HD)) for t in x.split(H * HD, -1)]


def loss_gpu(m, ids, target):
    x = training.embedding(ids, m.embedding.weight, scale=D ** 0.5)
    ly = m.layer
    q, k, v = heads(ly.qkv(recurrent.norm_conv1d(x, ly.norm, ly.conv)))
    o, state = recurrent.decay_attention(q, k, v, ly.log_decay, scale=HD ** -0.5)
    gn = ly.group_norm
    y = recurrent.group_norm_act(o.reshape(-1, H * HD), H, gn.weight, gn.bias, gn.eps, "silu").reshape(B, -1, H * HD)
    x = x + ly.out(y)
    return F.cross_entropy(F.linear(x, m.embedding.weight).flatten(0, 1), target.flatten()), state


def loss_ref(m, ids, target):
    x = m.embedding(ids) * D ** 0.5
    ly = m.layer
    # rows before the sequence are zeros before the norm
    h = ly.norm(F.pad(x, (0, 0, 3, 0)))
    h = F.conv1d(h.transpose(1, 2), ly.conv.weight, ly.conv.bias, groups=D).transpose(1, 2)
    q, k, v = heads(ly.qkv(h))
    o, state = recur(q, k, v, ly.log_decay, HD ** -0.5)
    y = F.silu(ly.group_norm(o.reshape(-1, H * HD))).reshape(B, -1, H * HD)
    x = x + ly.out(y)
    return F.cross_entropy(F.linear(x, m.embedding.weight).flatten(0, 1), target.flatten()), state


def test_training_step():
    """fp32: every gradient within 2^-24 * 64 * 64 of its norm (64 units for each of the operators' chains, some ten of
    which follow one another; LayerNorm and cross entropy divide by spreads of order one), and clipped alike."""
    ids, target = torch.randint(0, V, (B, L)), torch.randint(0, V, (B, L))
    ref = model().double()
    loss_ref(ref, ids, target)[0].backward()
    m = model().cuda()
    loss, _ = loss_gpu(m, ids.cuda(), target.cuda())
    loss.backward()
    norm = training.clip_grad_norm_(m.parameters(), 0.1)
    want = torch.nn.utils.clip_grad_norm_(ref.parameters(), 0.1)
    tol = 2.0 ** -24 * 64 * 64
    assert abs(float(norm) - float(want)) <= tol * float(want)
    for (name, a), b in zip(m.named_parameters(), ref.parameters()):
        assert (a.grad.double().cpu() - b.grad).norm() <= tol * b.grad.norm() + 1e-9, name
    ops.check_device()


def test_training_step_in_bf16_and_as_a_graph():
    """The same step in bf16, captured: replays give the eager gradients' bits."""
    m = model().cuda().bfloat16()
    m.layer.log_decay = m.layer.log_decay.float()
    ids, target = torch.randint(0, V, (B, L)).cuda(), torch.randint(0, V, (B, L)).cuda()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        grads = torch.autograd.grad(loss_gpu(m, ids, target)[0], list(m.parameters()))
        first = [g.clone() for g in grads]
        clipped = [torch.empty_like(g) for g in first]
        norm = ops.clip_grads(first, 0.1, out=clipped)
        del grads
        torch.cuda.synchronize()
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr, stream=side):
            again = list(torch.autograd.grad(loss_gpu(m, ids, target)[0], list(m.parameters())))
            n2 = ops.clip_grads(again, 0.1)
        gr.replay()
        torch.cuda.synchronize()
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(norm, n2) and all(torch.equal(a, b) for a, b in zip(clipped, again))


def test_prompt_then_tokens():
    """The attention of a prompt, then one token at a time, gives the whole sequence's outputs."""
    g = torch.Generator().manual_seed(2)
    table = torch.randn(V, 3 * H * HD, generator=g).cuda()
    ids = torch.randint(0, V, (B, L), generator=g).cuda()
    ld = torch.tensor([-0.02, -0.3]).cuda()
    q, k, v = heads(ops.embedding(ids, table))
    whole, end = ops.decay_attention(q, k, v, ld)
    o, state = ops.decay_attention(q[:, :50], k[:, :50], v[:, :50], ld)
    outs = [o]
    for t in range(50, L):
        qt, kt, vt = heads(ops.embedding(ids[:, t], table))
        outs.append(ops.decay_attention_step(qt, kt, vt, ld, state)[0].unsqueeze(1))
    assert (torch.cat(outs, 1) - whole).norm() <= 2.0 ** -24 * 64 * whole.norm() and (state - end).norm() <= 2.0 ** -24 * 64 * end.norm()


def test_the_lm_looks_its_rows_up():
    torch.manual_seed(3)
    lm = HdcMambaLM(100, 64, 1, 64, 1, chunk_size=64, use_model=False).cuda().bfloat16()
    ids = torch.randint(0, 100, (2, 64)).cuda()
    seen = []
    hook = lm.layers[0]._forward_inplace
    lm.layers[0]._forward_inplace = lambda h: (seen.append(h.clone()), hook(h))[1]
    with torch.no_grad():
        lm(ids)
    assert torch.equal(seen[0], lm.embedding.weight[ids])
    lm(ids).float().sum().backward()
    assert lm.embedding.weight.grad.isfinite().all()
