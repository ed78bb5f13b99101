"""The group norm stays inside the workspace that its size functions ask for, whatever the kernels
that a shape and type take."""
import ctypes

import pytest
import torch

from hdcmamba_b200 import _lib, ops

pytestmark = pytest.mark.gpu
DEV = "cuda"
P = ctypes.c_void_p


def rand(*shape, seed, dtype):
    return torch.randn(*shape, generator=torch.Generator(device=DEV).manual_seed(seed), device=DEV).to(dtype)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("N,S,C,G", [
    (3000, 1, 1024, 2), (700, 1, 1024, 1), (5, 1, 520, 1), (900, 1, 514, 1), (40, 1, 1032, 1), (300, 1, 768, 12),
    (33, 1, 4096, 1), (3, 1, 5000, 1), (2, 225, 96, 8), (2, 3000, 64, 4), (3, 40, 2048, 1), (2, 2, 3000, 3), (7, 9, 36, 3),
])
def test_workspace_is_enough(N, S, C, G, dtype):
    lib = _lib.load()
    x, dy = rand(N, S, C, seed=1, dtype=dtype), rand(N, S, C, seed=2, dtype=dtype)
    w, b = rand(C, seed=3, dtype=dtype), rand(C, seed=4, dtype=dtype)
    y, mean, rstd = ops.group_norm_act(x, G, w, b, act="silu", stats=True)
    dx, dw, db = ops.group_norm_act_bwd(dy, x, mean, rstd, G, w, b, act="silu")
    code = _lib.HDC_BF16 if dtype == torch.bfloat16 else _lib.HDC_F32
    stream = P(torch.cuda.current_stream().cuda_stream)

    def ptr(t):
        return P(t.data_ptr())

    def fenced(need):
        buf = torch.full((need + 65536,), 0xA5, device=DEV, dtype=torch.uint8)
        return buf, lambda: bool((buf[need:] == 0xA5).all())

    need = lib.hdc_group_norm_workspace_bytes(N, S, C, G)
    ws, whole = fenced(need)
    y2 = torch.empty_like(y)
    _lib.call("hdc_group_norm_fwd", code, code, ptr(x), S * C, C, ptr(w), ptr(b), ptr(y2), S * C, C, None, None, ptr(ws),
              need, N, S, C, G, 1e-5, _lib.HDC_ACT_SILU, stream)
    assert torch.equal(y2, y) and whole()
    need = lib.hdc_group_norm_bwd_workspace_bytes(N, S, C, G)
    ws, whole = fenced(need)
    out = [torch.empty_like(t) for t in (dx, dw, db)]
    _lib.call("hdc_group_norm_bwd", code, code, ptr(dy), S * C, C, ptr(x), S * C, C, ptr(mean), ptr(rstd), ptr(w), ptr(b),
              ptr(out[0]), S * C, C, ptr(out[1]), ptr(out[2]), ptr(ws), need, N, S, C, G, _lib.HDC_ACT_SILU, stream)
    assert all(torch.equal(a, c) for a, c in zip(out, (dx, dw, db))) and whole()
