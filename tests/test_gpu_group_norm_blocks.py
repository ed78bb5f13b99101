"""Group norm of channels that split into odd groups: blocks of whole groups that a wide load
divides would not fit an SM's shared memory, so such calls take narrower loads."""
import pytest
import torch

from test_gpu_group_norm_wide import BF16, F32, run_all

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("N,S", [(3, 1), (2, 5), (1, 130)])
@pytest.mark.parametrize("C,G", [(6152, 8), (6168, 8), (8200, 8), (8184, 2), (12300, 4), (6146, 2), (65520, 16)])
def test_odd_groups(C, G, N, S, dtype):
    run_all(N, S, C, G, dtype)
