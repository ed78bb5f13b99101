"""Sizes of the group norm's workspaces (computed on the host)."""
import pytest

from hdcmamba_b200 import _lib


def fwd(*shape):
    return _lib.load().hdc_group_norm_workspace_bytes(*shape)


def bwd(*shape):
    return _lib.load().hdc_group_norm_bwd_workspace_bytes(*shape)


@pytest.mark.parametrize("G", [1, 2, 4, 8, 16, 32])
def test_one_position_takes_one_set_of_sums_per_cta(G):
    """Groups that the one-pass kernel holds (up to 1024 channels here): a few CTAs per SM, whatever
    the number of samples; 4 of 2 x 148 at most, with 8 bytes per channel."""
    N, C = 32768, 1024
    assert fwd(N, 1, C, G) == 0
    assert 0 < bwd(N, 1, C, G) <= 296 * C * 8
    assert bwd(2 * N, 1, C, G) == bwd(N, 1, C, G)
    assert fwd(2 ** 21, 1, C, G) == 0 and bwd(2 ** 21, 1, C, G) <= 296 * C * 8


@pytest.mark.parametrize("N,S,C,G", [(8192, 1, 4096, 1), (4096, 1, 2056, 1), (4096, 3, 2048, 1), (512, 20, 6144, 2)])
def test_wide_groups_take_one_set_of_sums_per_sample(N, S, C, G):
    assert bwd(N, S, C, G) <= N * (C + G) * 8


def test_nothing_for_nothing():
    for shape in ((0, 1, 64, 4), (4, 0, 64, 4), (4, 1, 64, 5), (4, 1, 0, 1), (4, 1, 64, 0)):
        assert fwd(*shape) == 0 and bwd(*shape) == 0
