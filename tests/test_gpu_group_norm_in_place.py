"""The group norm's gradient may be written over x or over dy (hdc_group_norm_bwd)."""
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
@pytest.mark.parametrize("off", [0, 1])
@pytest.mark.parametrize("N,S,C,G", [
    (5000, 1, 512, 8), (700, 1, 1024, 1), (333, 1, 77, 7), (9, 1, 1500, 1), (3, 1, 5000, 1),  # one position
    (2, 225, 96, 8), (3, 77, 30, 3), (2, 4000, 64, 4), (1, 3000, 33, 3), (2, 40, 5000, 1),    # several
])
def test_dx_over_x_or_dy(N, S, C, G, off, dtype):
    """off: one column into rows of C + 1, so that loads are one by one."""
    lib = _lib.load()
    pitch = C + off

    def view(seed):
        return rand(N, S, pitch, seed=seed, dtype=dtype)[..., off:]

    w, b = rand(C, seed=3, dtype=dtype), rand(C, seed=4, dtype=dtype)
    x, dy = view(1), view(2)
    _, mean, rstd = ops.group_norm_act(x, G, w, b, act="silu", stats=True)
    want = ops.group_norm_act_bwd(dy, x, mean, rstd, G, w, b, act="silu")
    code = _lib.HDC_BF16 if dtype == torch.bfloat16 else _lib.HDC_F32
    need = lib.hdc_group_norm_bwd_workspace_bytes(N, S, C, G)
    ws = torch.empty(need, device=DEV, dtype=torch.uint8)
    for over in ("x", "dy"):
        x, dy = view(1), view(2)
        dx = x if over == "x" else dy
        dw, db = torch.empty_like(w), torch.empty_like(b)
        _lib.call("hdc_group_norm_bwd", code, code, P(dy.data_ptr()), dy.stride(0), dy.stride(1), P(x.data_ptr()),
                  x.stride(0), x.stride(1), P(mean.data_ptr()), P(rstd.data_ptr()), P(w.data_ptr()), P(b.data_ptr()),
                  P(dx.data_ptr()), dx.stride(0), dx.stride(1), P(dw.data_ptr()), P(db.data_ptr()), P(ws.data_ptr()),
                  need, N, S, C, G, _lib.HDC_ACT_SILU, P(torch.cuda.current_stream().cuda_stream))
        for a, c in zip((dx, dw, db), want):
            assert torch.equal(a, c), over
