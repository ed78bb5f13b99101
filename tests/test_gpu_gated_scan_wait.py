"""A wait between the tiles of a sequence that runs out: the call reports it and shows NaN, and the
calls after it are right.  The limit is set to 0, so that a tile gives up on the first result
that is not there yet; nothing hangs or faults."""
import pytest
import torch

from hdcmamba_b200 import _lib, ops

DEV = "cuda"


@pytest.fixture
def no_waiting():
    def limit(ns):
        _lib.call("hdc_gated_scan_wait_limit", ns)
    yield limit
    limit(2_000_000_000)
    torch.cuda.synchronize()
    _lib.load().hdc_device_error(1)


def test_limit_is_checked():
    with pytest.raises(_lib.HdcError, match="at most"):
        _lib.call("hdc_gated_scan_wait_limit", 2_000_000_001)


@pytest.mark.gpu
@pytest.mark.parametrize("backward", [False, True])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_wait_that_runs_out(dtype, backward, no_waiting):
    B, L, ds = 2, 32768, 64
    g = torch.Generator(device=DEV).manual_seed(1)
    projs = torch.randn(B, L, 3 * ds, generator=g, device=DEV).to(dtype)
    dy = torch.randn(B, L, ds, generator=g, device=DEV).to(dtype)
    A_log = torch.zeros(ds, device=DEV)
    ops.check_device()

    def run(states=[None]):
        if not backward:
            y, h, states[0] = ops.gated_scan(projs, A_log, ds, return_states=True)
            return y, h
        if states[0] is None:
            states[0] = ops.gated_scan(projs, A_log, ds, return_states=True)[2]
        dp, dA, dh0 = ops.gated_scan_bwd(dy, projs, A_log, states[0], ds, need_dh0=True)
        return dp, dA, dh0

    want = run()
    assert all(bool(torch.isfinite(t).all()) for t in want)
    for _ in range(10):  # a tile that finds all that it needs gives up on nothing
        no_waiting(0)
        got = run()
        no_waiting(2_000_000_000)
        after = run()  # not cleared in between: what ran out before does not reach this call
        torch.cuda.synchronize()
        if bool(got[0].isnan().any()):
            break
    nan = got[0].isnan()
    assert bool(nan.any())
    assert torch.equal(got[0][~nan], want[0][~nan])  # wrong values are never finite
    assert all(torch.equal(a, b) for a, b in zip(after, want))
    with pytest.raises(_lib.HdcError, match="61"):
        ops.check_device()
    ops.check_device()  # cleared
