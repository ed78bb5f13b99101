"""GatedRecurrentBlock: training, prefill and decode through the operators together."""
import pytest
import torch
import torch.nn.functional as F

from hdcmamba_b200 import _lib
from hdcmamba_b200.recurrent import GatedRecurrentBlock
from recurrent_ref import norm_values, scan_values

pytestmark = pytest.mark.gpu
DEV = "cuda"


def block(dtype=torch.float32, d_model=64, d_state=48, heads=4):
    torch.manual_seed(3)
    return GatedRecurrentBlock(d_model, d_state, heads).to(DEV).to(dtype)


def plain(blk, x, reset=None):
    """The layer's definition on its own parameters, in 64 bits (differentiable)."""
    p = {k: v.detach().double().requires_grad_() for k, v in blk.named_parameters()}
    x = x.double()
    h = F.layer_norm(F.pad(x, (0, 0, 3, 0)), (blk.d_model,), p["norm.weight"], p["norm.bias"], blk.norm.eps)
    h = F.conv1d(h.transpose(1, 2), p["conv1d.weight"], p["conv1d.bias"], groups=blk.d_model).transpose(1, 2)
    y = scan_values(F.linear(h, p["in_proj.weight"], p["in_proj.bias"]), p["A_log"], blk.d_state, None, reset)
    B, L, ds = y.shape
    z = norm_values(y.reshape(B * L, 1, ds), blk.num_heads, p["group_norm.weight"], p["group_norm.bias"],
                    blk.group_norm.eps, "silu").reshape(B, L, ds)
    return x + F.linear(z, p["out_proj.weight"]), p


def test_forward_and_gradients():
    """fp32 against 64 bits: 1e-4 of each result's largest value (cuBLAS fp32 products of depth
    64 and the norm of a state that starts near zero amplify 2^-24 by at most some hundreds)."""
    blk = block()
    x = torch.randn(2, 140, 64, generator=torch.Generator(device=DEV).manual_seed(1), device=DEV)
    reset = torch.zeros(2, 140, dtype=torch.bool, device=DEV)
    reset[1, 60] = True
    dy = torch.randn(2, 140, 64, generator=torch.Generator(device=DEV).manual_seed(2), device=DEV)
    y = blk(x, reset=reset)
    names = ["A_log", "in_proj.weight", "in_proj.bias", "group_norm.weight", "group_norm.bias", "out_proj.weight"]
    grads = torch.autograd.grad(y, [dict(blk.named_parameters())[n] for n in names], dy)
    want, p = plain(blk, x, reset)
    wgrads = torch.autograd.grad(want, [p[n] for n in names], dy.double())
    assert float((y.detach().double() - want.detach()).abs().max() / want.detach().abs().max()) < 1e-4
    for n, a, b in zip(names, grads, wgrads):
        assert float((a.double() - b).abs().max() / b.abs().max()) < 1e-3, n


@pytest.mark.parametrize("dtype,tol", [(torch.float32, 1e-4), (torch.bfloat16, 4e-2)])
@pytest.mark.parametrize("L0", [1, 2, 150])
def test_decode_continues_the_prefill(dtype, tol, L0):
    """Prefill of L0 rows and T steps equal the forward of L0 + T rows (bf16: the roundings of
    each row are the same up to the last places of the fp32 sums before them)."""
    blk = block(dtype)
    T = 12
    x = torch.randn(2, L0 + T, 64, generator=torch.Generator(device=DEV).manual_seed(1), device=DEV).to(dtype)
    with torch.no_grad():
        full = blk(x)
    y, st = blk.prefill(x[:, :L0])
    outs = [blk.step(x[:, L0 + t], st) for t in range(T)]
    got = torch.cat([y, torch.stack(outs, 1)], 1)
    assert float((got.float() - full.float()).abs().max() / full.float().abs().max()) < tol
    assert _lib.load().hdc_device_error(1) == 0


def test_training_follows_the_definition():
    """Gradient descent through the kernels in fp32 and through the definition in 64 bits: the
    same losses, step after step (each gradient is within 1e-3, the first test's bound, and five
    steps of rate 0.05 move the loss by well under its size)."""
    names = ["A_log", "in_proj.weight", "in_proj.bias", "group_norm.weight", "group_norm.bias", "out_proj.weight"]
    x = torch.randn(2, 140, 64, generator=torch.Generator(device=DEV).manual_seed(1), device=DEV)
    target = torch.roll(x, 1, 1)
    blk, ref = block(), block()
    for _ in range(5):
        loss = (blk(x) - target).square().mean()
        y, p = plain(ref, x)
        want = (y - target.double()).square().mean()
        assert abs(loss.item() - want.item()) < 1e-3 * want.item()
        mine = dict(blk.named_parameters())
        for mod, grads in ((blk, torch.autograd.grad(loss, [mine[n] for n in names])),
                           (ref, torch.autograd.grad(want, [p[n] for n in names]))):
            with torch.no_grad():
                for n, g in zip(names, grads):
                    dict(mod.named_parameters())[n].sub_(0.05 * g.float())


def test_library_kernels_ran():
    blk = block(torch.bfloat16)
    x = torch.randn(2, 64, 64, device=DEV).bfloat16().requires_grad_()
    n = _lib.launch_count()
    blk(x).float().sum().backward()
    assert _lib.launch_count() - n >= 6


def test_cpu_input_raises():
    with pytest.raises(RuntimeError, match="CUDA"):
        block()(torch.randn(1, 8, 64))
