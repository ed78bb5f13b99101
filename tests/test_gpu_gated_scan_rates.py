"""The gated recurrence at decay rates past fp32's range: A = -exp(A_log) is -inf in fp32, and a
step forgets the state at once."""
import pytest
import torch

from hdcmamba_b200 import ops
from recurrent_ref import check, scan_ref

pytestmark = pytest.mark.gpu
DEV = "cuda"


def rand(*shape, seed, dtype=torch.float32):
    return torch.randn(*shape, generator=torch.Generator(device=DEV).manual_seed(seed), device=DEV).to(dtype)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("L", [1, 9, 64, 70, 200])
@pytest.mark.parametrize("A_log", [80.0, 88.8, 100.0])
def test_rates_past_the_range(A_log, L, dtype):
    """The decays are 0 in 64 bits too, so outputs and gradients are each step's own."""
    B, ds = 2, 40
    projs = rand(B, L, 3 * ds, seed=1).to(dtype)
    a = torch.full((ds,), A_log, device=DEV)
    a[::2] = 0.0  # ordinary channels beside them
    h0, dy, dh = rand(B, ds, seed=2), rand(B, L, ds, seed=3).to(dtype), rand(B, ds, seed=4)
    ref = scan_ref(projs, a, ds, h0, None, dy, dh)
    y, h, st = ops.gated_scan(projs, a, ds, h0=h0, return_states=True)
    check(y, ref["y"], "y")
    check(h, ref["h_last"], "h_last")
    dp, dA, dh0 = ops.gated_scan_bwd(dy, projs, a, st, ds, dh_last=dh, need_dh0=True)
    check(dp, ref["dprojs"], "dprojs")
    check(dh0, ref["dh0"], "dh0")
    check(dA, ref["dA_log"], "dA_log")
    hs = h0.clone()
    for t in range(min(L, 3)):
        yt, _ = ops.gated_step(projs[:, t], a, hs, ds)
        check(yt, (ref["y"][0][:, t], ref["y"][1][:, t]), "step")
    nan = torch.full((ds,), float("nan"), device=DEV)
    assert bool(ops.gated_scan(projs, nan, ds, h0=h0)[0].isnan().all())
