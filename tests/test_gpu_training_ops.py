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


def test_two_threads_at_once():
    """Calls from two host threads on streams of their own."""
    import threading
    g = torch.Generator().manual_seed(4)
    q = torch.randn(2, 300, 2, 64, generator=g).cuda().bfloat16()
    ld = torch.tensor([-0.02, -0.3]).cuda()
    ids = torch.randint(0, V, (5000,), generator=g).cuda()
    dy = torch.randn(5000, 64, generator=g).cuda()
    xs = [torch.randn(9999, generator=g).cuda() for _ in range(3)]
    torch.cuda.synchronize()

    def work():
        s = torch.cuda.Stream()
        with torch.cuda.stream(s):
            for _ in range(20):
                leaf = q.clone().requires_grad_()
                o, e = recurrent.decay_attention(leaf, q, q, ld)
                r = [o.detach(), e.detach(), *torch.autograd.grad(o, [leaf], q), ops.embedding_bwd(dy, ids, V), ops.clip_grads(xs, None)]
        s.synchronize()
        return r

    want, got = work(), [None, None]

    def run(i):
        got[i] = work()

    threads = [threading.Thread(target=run, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for r in got:
        assert r is not None and all(torch.equal(a, b) for a, b in zip(want, r))


def test_refusals_of_the_library_raise():
    from hdcmamba_b200 import _lib
    x = torch.ones(100, device="cuda")
    for grads, out in (([x, x], None), ([x[:60], x[50:]], None), ([x[:50], x[50:]], [x[50:], x[:50]])):
        with pytest.raises(_lib.HdcError, match="overlaps"):
            ops.clip_grads(grads, 1.0, out=out)
    with pytest.raises(_lib.HdcError, match="max_norm"):
        ops.clip_grads([x], -1.0)
    q = torch.zeros(1, 4, 2, 8, device="cuda")
    with pytest.raises(_lib.HdcError, match="overlap"):
        ops.decay_attention(q, q, q, torch.zeros(2, device="cuda"), out=q[:, :1].expand(1, 4, 2, 8))
    with pytest.raises(RuntimeError, match="CPU"):
        ops.decay_attention(q, q.cpu(), q, torch.zeros(2, device="cuda"))
    with pytest.raises(RuntimeError, match="CPU"):
        ops.embedding(torch.zeros(3, dtype=torch.int64), q[0, 0])
    assert (x == 1).all()


def test_a_sequence_of_a_quarter_million_tokens():
    """Against two halves of it, joined by the state: the same bounds as for the definition (two roundings to bf16)."""
    g = torch.Generator().manual_seed(5)
    L = 262144 + 37
    q, k, v = (torch.randn(1, L, 1, 64, generator=g).cuda().bfloat16() for _ in range(3))
    ld = torch.tensor([-0.0005]).cuda()
    o, e = ops.decay_attention(q, k, v, ld, 0.1)
    cut = 100001
    a, m = ops.decay_attention(q[:, :cut], k[:, :cut], v[:, :cut], ld, 0.1)
    b, n = ops.decay_attention(q[:, cut:], k[:, cut:], v[:, cut:], ld, 0.1, m)
    both = torch.cat([a, b], 1).float()
    assert (o.float() - both).norm() <= 2 * 2 * 2 ** -8 * both.norm()
    assert (e - n).norm() <= 2 * 64 * 2.0 ** -24 * n.norm()
