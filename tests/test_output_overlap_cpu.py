"""Outputs whose rows overlap one another are refused before any CUDA call: two CTAs would write the
same memory.  (Inputs may overlap.)"""
import ctypes

import pytest

from hdcmamba_b200 import _lib

P = ctypes.c_void_p
E_SHAPE = -2
BIG = 1 << 40


def scan_fwd(sb, st, B=2, L=4, ds=8):
    return _lib.load().hdc_gated_scan_fwd(1, 0, P(16), 96, 24, P(16), None, None, P(16), sb, st, P(16), None, P(16), BIG,
                                          B, L, ds, None)


def scan_bwd(sb, st, B=2, L=4, ds=8):
    return _lib.load().hdc_gated_scan_bwd(1, 0, P(16), 96, 24, P(16), P(16), None, P(16), 32, 8, None, P(16), sb, st,
                                          P(16), None, P(16), BIG, B, L, ds, None)


def norm_fwd(sn, ss, N=2, S=3, C=8):
    return _lib.load().hdc_group_norm_fwd(1, 1, P(16), 24, 8, P(16), P(16), P(16), sn, ss, P(16), P(16), P(16), BIG, N, S,
                                          C, 2, 1e-5, 1, None)


def norm_bwd(sn, ss, N=2, S=3, C=8):
    return _lib.load().hdc_group_norm_bwd(1, 1, P(16), 24, 8, P(16), 24, 8, P(16), P(16), P(16), P(16), P(16), sn, ss,
                                          P(16), P(16), P(16), BIG, N, S, C, 2, 1, None)


@pytest.mark.parametrize("call", [
    lambda: scan_fwd(0, 8), lambda: scan_fwd(31, 8), lambda: scan_fwd(32, 7), lambda: scan_fwd(8, 8),
    lambda: scan_fwd(-32, 8), lambda: scan_fwd(7, 8, L=1), lambda: scan_fwd(7, 16),
    lambda: scan_bwd(0, 24), lambda: scan_bwd(95, 24), lambda: scan_bwd(96, 23), lambda: scan_bwd(23, 48),
    lambda: norm_fwd(0, 8), lambda: norm_fwd(23, 8), lambda: norm_fwd(24, 7), lambda: norm_fwd(24, 0, N=1),
    lambda: norm_fwd(4, 0, S=1), lambda: norm_bwd(0, 8), lambda: norm_bwd(23, 8), lambda: norm_bwd(24, 0),
])
def test_overlapping_outputs_are_refused(call):
    assert call() == E_SHAPE
    assert b"overlap" in _lib.load().hdc_error_string()
