"""Views as outputs of the gated recurrence: any that lie apart, in either order of batch and time;
expanded ones are refused."""
import pytest
import torch

from hdcmamba_b200 import _lib, ops

pytestmark = pytest.mark.gpu
DEV = "cuda"


def test_views_that_lie_apart_and_views_that_do_not():
    B, L, ds = 3, 150, 48
    g = torch.Generator(device=DEV).manual_seed(1)
    projs = torch.randn(B, L, 3 * ds, generator=g, device=DEV)
    dy = torch.randn(B, L, ds, generator=g, device=DEV)
    A_log = torch.zeros(ds, device=DEV)
    y, _, st = ops.gated_scan(projs, A_log, ds, return_states=True)
    dp = ops.gated_scan_bwd(dy, projs, A_log, st, ds)[0]
    for shape, order in (((L, B), (1, 0)), ((B, L), (0, 1))):
        out = torch.zeros(*shape, 2 * ds, device=DEV).permute(*order, 2)[..., 5:5 + ds]
        assert torch.equal(ops.gated_scan(projs, A_log, ds, out=out)[0], y)
        out = torch.zeros(*shape, 4 * ds, device=DEV).permute(*order, 2)
        assert torch.equal(ops.gated_scan_bwd(dy, projs, A_log, st, ds, out=out)[0][..., :3 * ds], dp)
    with pytest.raises(_lib.HdcError, match="overlap"):
        ops.gated_scan(projs, A_log, ds, out=torch.zeros(1, L, ds, device=DEV).expand(B, L, ds))
    with pytest.raises(_lib.HdcError, match="overlap"):
        ops.gated_scan_bwd(dy, projs, A_log, st, ds, out=torch.zeros(1, L, 3 * ds, device=DEV).expand(B, L, 3 * ds))
    one = torch.zeros(1, ds, device=DEV).expand(B, ds)
    with pytest.raises(_lib.HdcError, match="overlap"):
        ops.gated_step(projs[:, 0], A_log, torch.zeros(B, ds, device=DEV), ds, out=one)
    with pytest.raises(ValueError, match="h_out"):
        ops.gated_step(projs[:, 0], A_log, torch.zeros(B, ds, device=DEV), ds, h_out=one)


def test_nothing_to_write_is_nothing_to_refuse():
    B, ds = 2, 8
    A_log, h0 = torch.zeros(ds, device=DEV), torch.ones(B, ds, device=DEV)
    none = torch.zeros(B, 0, 3 * ds, device=DEV)
    out = torch.zeros(1, 0, ds, device=DEV).expand(B, 0, ds)
    assert torch.equal(ops.gated_scan(none, A_log, ds, h0=h0, out=out)[1], h0)
