"""The trainable LN + conv of ``GatedRecurrentBlock``: every gradient is the derivative of the
layer's own forward, the norm bias and the rows before the sequence included, against the
definition in 64 bits."""
import pytest
import torch
import torch.nn.functional as F

from hdcmamba_b200 import _lib, ops
from hdcmamba_b200.recurrent import GatedRecurrentBlock, norm_conv1d
from recurrent_ref import norm_values, scan_values

pytestmark = pytest.mark.gpu
DEV = "cuda"


def rand(*shape, seed, dtype=torch.float32):
    return torch.randn(*shape, generator=torch.Generator(device=DEV).manual_seed(seed), device=DEV).to(dtype)


def block(bias):
    """A layer whose norm bias and other parameters have left their initial values."""
    torch.manual_seed(3)
    blk = GatedRecurrentBlock(64, 48, 4).to(DEV)
    with torch.no_grad():
        blk.norm.bias.copy_(bias * rand(64, seed=21))
        blk.norm.weight.add_(0.2 * rand(64, seed=22))
        blk.conv1d.bias.copy_(0.1 * rand(64, seed=23))
        blk.conv1d.weight.add_(0.2 * rand(64, 1, 4, seed=24))
    return blk


def plain(blk, x, reset=None):
    """The layer's definition on its own parameters, in 64 bits."""
    p = {k: v.detach().double().requires_grad_() for k, v in blk.named_parameters()}
    h = F.layer_norm(F.pad(x, (0, 0, 3, 0)), (blk.d_model,), p["norm.weight"], p["norm.bias"], blk.norm.eps)
    h = F.conv1d(h.transpose(1, 2), p["conv1d.weight"], p["conv1d.bias"], groups=blk.d_model).transpose(1, 2)
    y = scan_values(F.linear(h, p["in_proj.weight"], p["in_proj.bias"]), p["A_log"], blk.d_state, None, reset)
    B, L, ds = y.shape
    z = norm_values(y.reshape(B * L, 1, ds), blk.num_heads, p["group_norm.weight"], p["group_norm.bias"],
                    blk.group_norm.eps, "silu").reshape(B, L, ds)
    return x + F.linear(z, p["out_proj.weight"]), p


@pytest.mark.parametrize("L", [1, 2, 3, 140])
@pytest.mark.parametrize("bias", [0.0, 0.02, 0.5])
def test_every_gradient_of_the_block(bias, L):
    """Within 1e-3 of each gradient's largest value: products of depth 64 and the norm of a state
    that starts near zero amplify 2^-24 by at most some hundreds; statistics held in 16 bits, 2^-9,
    or a left-out term would not pass."""
    blk = block(bias)
    x = rand(2, L, 64, seed=1).requires_grad_()
    dy = rand(2, L, 64, seed=2)
    names = [n for n, _ in blk.named_parameters()]
    grads = torch.autograd.grad(blk(x), [x] + list(blk.parameters()), dy)
    x64 = x.detach().double().requires_grad_()
    want, p = plain(blk, x64)
    wgrads = torch.autograd.grad(want, [x64] + [p[n] for n in names], dy.double())
    for n, a, b in zip(["x"] + names, grads, wgrads):
        assert a.shape == b.shape
        assert float((a.double() - b).abs().max()) <= 1e-3 * float(b.abs().max()), n


def conv_ref(x, nw, nb, cw, cb, dy):
    """The definition's output and gradients by autograd in 64 bits."""
    leaves = [t.double().requires_grad_() for t in (x, nw, nb, cw, cb)]
    n = F.layer_norm(F.pad(leaves[0], (0, 0, 3, 0)), (x.shape[2],), leaves[1], leaves[2], 1e-5)
    y = F.conv1d(n.transpose(1, 2), leaves[3].unsqueeze(1), leaves[4], groups=x.shape[2]).transpose(1, 2)
    return y.detach(), torch.autograd.grad(y, leaves, dy.double())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("B,L,D", [(1, 1, 8), (2, 2, 8), (3, 3, 64), (2, 4, 24), (1, 7, 768), (2, 16, 40), (3, 145, 1024),
                                   (9, 300, 256), (1, 4097, 64), (2, 33, 2048)])
def test_operator_against_64_bits(B, L, D, dtype):
    """Rounding: the row statistics and sums of depth D have errors of at most 64 units of 2^-24 with
    random signs, each gradient a sum of terms off by some 16 units more, sums over n rows n/32
    more; a unit is the largest term (row: of dx, channel: of the sum's absolute values) and the
    norm's backward multiplies by rstd |n| < 8.  bf16 results add half a unit in the last place."""
    x = (rand(B, L, D, seed=1) + 0.3 * rand(D, seed=2)).to(dtype)
    nw, nb = (1 + 0.2 * rand(D, seed=3)).to(dtype), (0.5 * rand(D, seed=4)).to(dtype)
    cw, cb = (0.5 * rand(D, 4, seed=5)).to(dtype), (0.1 * rand(D, seed=6)).to(dtype)
    dy = rand(B, L, D, seed=7, dtype=dtype)
    y, mean, rstd = ops.ln_conv_train(x, nw, nb, cw, cb)
    want, grads = conv_ref(x, nw, nb, cw, cb, dy)
    half = 2.0 ** -8 if dtype == torch.bfloat16 else 2.0 ** -23
    unit = (16 + 64) * 8 * 2.0 ** -24
    assert mean.dtype == rstd.dtype == torch.float32
    x64 = x.double()
    torch.testing.assert_close(mean.double(), x64.mean(-1), rtol=0, atol=64 * 2.0 ** -24)
    torch.testing.assert_close(rstd.double(), (x64.var(-1, correction=0) + 1e-5).rsqrt(), rtol=256 * 2.0 ** -24, atol=0)
    assert bool(((y.double() - want).abs() <= half * want.abs() + unit * want.abs().max()).all())
    got = ops.ln_conv_train_bwd(dy, x, mean, rstd, nw, nb, cw)
    dn = dy.double().abs().sum((0, 1))  # of each channel: |n| < 8, |conv weight| < 3
    for name, a, b in zip(("dx", "dnw", "dnb", "dcw", "dcb"), got, grads):
        if name == "dx":
            size = b.abs().amax(-1, keepdim=True)
        else:
            size = 3 * (1 + B * L / 32 / 80) * (dn.unsqueeze(1) if name == "dcw" else dn)
        assert a.dtype == dtype
        assert bool(((a.double() - b).abs() <= half * b.abs() + unit * size).all()), name


def test_operator_against_differences():
    """Directional derivatives by central differences of the definition in 64 bits (step 1e-6); the
    fp32 gradient's rounding, 1e-5 of the terms' size, decides."""
    B, L, D = 2, 11, 16
    p = [rand(B, L, D, seed=1), 1 + 0.2 * rand(D, seed=3), 0.5 * rand(D, seed=4), 0.5 * rand(D, 4, seed=5),
         0.1 * rand(D, seed=6)]
    dy = rand(B, L, D, seed=7)
    _, mean, rstd = ops.ln_conv_train(*p)
    grads = ops.ln_conv_train_bwd(dy, p[0], mean, rstd, *p[1:4])
    for i, gr in enumerate(grads):
        for seed in range(3):
            v = rand(*gr.shape, seed=100 + seed).double()
            ends = []
            for step in (1e-6, -1e-6):
                q = [t.double() for t in p]
                q[i] = q[i] + step * v
                n = F.layer_norm(F.pad(q[0], (0, 0, 3, 0)), (D,), q[1], q[2], 1e-5)
                y = F.conv1d(n.transpose(1, 2), q[3].unsqueeze(1), q[4], groups=D).transpose(1, 2)
                ends.append(float((y * dy.double()).sum()))
            size = float((gr.double() * v).abs().sum())
            assert abs(float((gr.double() * v).sum()) - (ends[0] - ends[1]) / 2e-6) <= 1e-5 * size + 1e-6, (i, seed)


def test_the_drop_in_keeps_the_references_formulas():
    """hdc_ln_conv_bwd: the norm bias and the rows before the sequence stay left out."""
    B, L, D = 2, 40, 64
    x, dy = rand(B, L, D, seed=1), rand(B, L, D, seed=7)
    nw, nb = 1 + 0.2 * rand(D, seed=3), 0.5 * rand(D, seed=4)
    cw, cb = 0.5 * rand(D, 4, seed=5), 0.1 * rand(D, seed=6)
    _, mean, rstd = ops.ln_conv(x, nw, nb, cw, cb, stats=True)
    old = ops.ln_conv_bwd(dy, x, mean, rstd, nw, cw)
    _, m32, r32 = ops.ln_conv_train(x, nw, nb, cw, cb)
    new = ops.ln_conv_train_bwd(dy, x, m32, r32, nw, nb, cw)
    pads = sum(dy[:, s].sum(0) * cw[:, :3 - s].sum(1) for s in range(3))  # dn of the rows -3 .. -1
    torch.testing.assert_close(new[2] - old[2], pads, rtol=1e-4, atol=1e-4)
    # the bf16 statistics are off by 2^-9 of |n| < 8, which a sum of 80 terms of random sign passes on
    torch.testing.assert_close(new[3] - old[3], (nb * dy.sum((0, 1))).unsqueeze(1).expand(D, 4), rtol=0.05, atol=0.5)


def test_other_layouts_and_types():
    """Strided x and dy, parameters of another type, no gradient asked for."""
    blk = block(0.3)
    x = rand(64, 30, 4, seed=1).permute(2, 1, 0)
    dy = rand(64, 30, 4, seed=2).permute(2, 1, 0)
    p = list(blk.norm.parameters()) + list(blk.conv1d.parameters())
    y = norm_conv1d(x, blk.norm, blk.conv1d)
    again = norm_conv1d(x.contiguous(), blk.norm, blk.conv1d)
    assert torch.equal(y, again)
    for a, b in zip(torch.autograd.grad(y, p, dy), torch.autograd.grad(again, p, dy.contiguous())):
        assert torch.equal(a, b)
    low = norm_conv1d(x.bfloat16(), blk.norm, blk.conv1d)
    assert low.dtype == torch.bfloat16
    assert all(g.dtype == torch.float32 for g in torch.autograd.grad(low, p, dy.bfloat16()))
    with torch.no_grad():
        assert torch.equal(norm_conv1d(x, blk.norm, blk.conv1d), y)


def test_refusals():
    blk = block(0.3)
    x = rand(2, 5, 64, seed=1).requires_grad_()
    with pytest.raises(RuntimeError, match="once"):
        torch.autograd.grad(norm_conv1d(x, blk.norm, blk.conv1d).sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="CUDA"):
        norm_conv1d(x.cpu(), blk.norm, blk.conv1d)
    nw, nb, cw, cb = (torch.zeros(s, device=DEV) for s in (64, 64, (64, 4), 64))
    out, mean, rstd = ops.ln_conv_train(x.detach(), nw, nb, cw, cb)
    with pytest.raises(ValueError, match="mean"):
        ops.ln_conv_train_bwd(out, x.detach(), mean.bfloat16(), rstd, nw, nb, cw)
    with pytest.raises(ValueError, match="shape"):
        ops.ln_conv_train_bwd(out[:, :4], x.detach(), mean, rstd, nw, nb, cw)
    with pytest.raises(TypeError, match="mismatch"):
        ops.ln_conv_train_bwd(out.bfloat16(), x.detach(), mean, rstd, nw, nb, cw)
    with pytest.raises(TypeError, match="dtype"):
        ops.ln_conv_train(x.detach().half(), nw, nb, cw, cb)
    with pytest.raises(_lib.HdcError, match="multiple"):
        ops.ln_conv_train(torch.zeros(1, 4, 6, device=DEV), nw[:6], nb[:6], cw[:6], cb[:6])
