"""Sequences long enough that the exchange between tiles goes through its coarser entries (spans
of 16 tiles, 1024 steps; links of 16 spans, 16384 steps), with gates that remember across them,
against the definition in 64 bits."""
import pytest
import torch

from hdcmamba_b200 import ops
from recurrent_ref import check, scan_ref

pytestmark = pytest.mark.gpu
DEV = "cuda"
F32, BF16 = torch.float32, torch.bfloat16


def rand(*shape, seed, dtype=F32):
    return torch.randn(*shape, generator=torch.Generator(device=DEV).manual_seed(seed), device=DEV).to(dtype)


def inputs(B, L, ds, dtype, centre):
    projs = rand(B, L, 3 * ds, seed=1)
    projs[..., :ds] = centre + 0.5 * projs[..., :ds]
    return projs.to(dtype), torch.log(torch.linspace(0.5, 1.5, ds, device=DEV))


def run_all(projs, A_log, ds, reset):
    B, L = projs.shape[:2]
    h0, dh = 30 * rand(B, ds, seed=3), 30 * rand(B, ds, seed=8)
    dy = rand(B, L, ds, seed=7, dtype=projs.dtype)
    y, h, st = ops.gated_scan(projs, A_log, ds, h0=h0, reset=reset, return_states=True)
    dp, dA, dh0 = ops.gated_scan_bwd(dy, projs, A_log, st, ds, reset=reset, dh_last=dh, need_dh0=True)
    ref = scan_ref(projs, A_log, ds, h0, reset, dy, dh)
    for k, v in {"y": y, "h_last": h, "dprojs": dp, "dA_log": dA, "dh0": dh0}.items():
        check(v, ref[k], k)
    return ref


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("resets", [False, True])
@pytest.mark.parametrize("L", [1023, 1024, 1025, 5000, 16383, 16384, 16385, 17500, 33000])
def test_memory_across_spans_and_links(L, resets, dtype):
    """softplus(-9.5) is 7e-5, so that a state still holds exp(-2.5) of itself after 33000 steps: a
    wrong span or link shows at full size."""
    B, ds = 2, 6
    projs, A_log = inputs(B, L, ds, dtype, -9.5)
    reset = None
    if resets:  # one or two documents per link, at no tile's border
        reset = torch.zeros(B, L, dtype=torch.bool, device=DEV)
        reset[0, L // 3] = True
        reset[1, [5, 2 * L // 3]] = True
    ref = run_all(projs, A_log, ds, reset)
    if not resets:  # the carried state reaches the end, the carried gradient the start
        none = scan_ref(projs, A_log, ds, None)
        assert float((ref["h_last"][0] - none["h_last"][0]).abs().max()) > 1.0


@pytest.mark.parametrize("resets", [False, True])
@pytest.mark.parametrize("ds", [601, 1000, 512, 640])
def test_wide_tiles_partly_empty(ds, resets):
    """bf16 tiles of 128 channels whose last one is not full (and full ones)."""
    B, L = 2, 1300
    projs, A_log = inputs(B, L, ds, BF16, -6.0)
    reset = None
    if resets:
        reset = rand(B, L, seed=5) > 2.5
    run_all(projs, A_log, ds, reset)
