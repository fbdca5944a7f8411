"""Waits of the chunk kernel that run out at every depth of its pipeline, over operands laid out once: what is on its way
is waited for, and the call is computed again."""

from __future__ import annotations

import pytest
import torch

from tests.test_gpu_paged_attention import Batch
from tricast_b200 import _native as N

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("polls", [0, 1, 2, 3, 5, 8, 13, 40, 100])
@pytest.mark.parametrize("scheme", ["fp8_row", "mxfp4"])
def test_limits_of_few_polls(scheme, polls):
    b = Batch([150, 1, 130], [900, 40, 700], 8, 1, 128, 16, scheme, torch.bfloat16)
    N.lib().tc_set_wait_limit(polls)
    try:
        for _ in range(3):
            b.check()
    finally:
        N.lib().tc_set_wait_limit(-1)
    b.check()
