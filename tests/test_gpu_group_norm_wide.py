"""Group norm of wide groups: every number of channels per group that the header allows launches
in both directions, at one position and at several."""
import pytest
import torch

from hdcmamba_b200 import ops
from recurrent_ref import check, norm_ref

pytestmark = pytest.mark.gpu
DEV = "cuda"
F32, BF16 = torch.float32, torch.bfloat16


def rand(*shape, seed, dtype=F32):
    return torch.randn(*shape, generator=torch.Generator(device=DEV).manual_seed(seed), device=DEV).to(dtype)


def run_all(N, S, C, G, dtype):
    x = (rand(N, S, C, seed=1) + 0.3 * rand(C, seed=2)).to(dtype)
    w, b = (1 + 0.2 * rand(C, seed=3)).to(dtype), (0.3 * rand(C, seed=4)).to(dtype)
    dy = rand(N, S, C, seed=5, dtype=dtype)
    y, mean, rstd = ops.group_norm_act(x, G, w, b, act="silu", stats=True)
    dx, dw, db = ops.group_norm_act_bwd(dy, x, mean, rstd, G, w, b, act="silu")
    ref = norm_ref(x, G, w, b, 1e-5, "silu", dy)
    for k, v in {"y": y, "mean": mean, "dx": dx, "dw": dw, "db": db}.items():
        check(v, ref[k], k)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("N,S", [(3, 1), (2, 3), (2, 70)])
@pytest.mark.parametrize("Cg,G", [(3072, 1), (3073, 1), (3080, 2), (4095, 1), (4096, 1), (4096, 2), (4097, 1)])
def test_group_widths(Cg, G, N, S, dtype):
    """Around the widths at which a step's shared memory and its kernel change."""
    run_all(N, S, Cg * G, G, dtype)
