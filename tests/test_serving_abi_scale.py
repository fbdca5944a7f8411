"""CPU check: a softmax scale that is finite but not so once the kernels' factor log2(e) is in it is refused."""

from __future__ import annotations

import pytest

from tests.test_serving_abi import P, _cache
from tricast_b200 import _native as N


@pytest.mark.parametrize("scale", [3e38, -3e38, float("inf"), float("nan")])
def test_scales_beyond_fp32_are_refused(scale):
    lib = N.lib()
    assert lib.tc_paged_attention(_cache(), P, 256, 64, 2, 4, P, 1, 1, P, P, 1, 2, scale, 1, 0, P, None, None, 0,
                                  None) == N.TC_INVALID_ARGUMENT
    assert b"scale" in lib.tc_last_error()
