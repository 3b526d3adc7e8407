"""Channels-last group norms at the number of channels where a run of pixels fills the LDS that a launch may have: 8192 values of eight bytes."""
import pytest

import norm_dense_muon as R  # noqa: F401 - the helpers below use it
from test_gpu_norm_dense_muon import _check_norm, _check_norm_grad, _norm_case

pytestmark = pytest.mark.gpu


# c, groups: a group per channel up to the limit and beyond it, odd numbers, few groups, groups that a workgroup holds
@pytest.mark.parametrize("c,groups", [(7904, 7904), (7905, 7905), (8191, 8191), (8192, 8192), (8192, 4096), (8192, 1), (8192, 128), (8188, 2047), (8193, 8193), (8196, 4)])
@pytest.mark.parametrize("n,h,w", [(2, 3, 5), (1, 9, 16)], ids=str)
def test_channels_last(n, h, w, c, groups):
    x, scale, bias, dy = _norm_case(n, c, h, w, True, c + groups)
    _check_norm(x, scale, bias, groups, "gelu", True)
    _check_norm_grad(dy, x, scale, bias, groups, "silu", True)
