"""Windows and token bounds beyond 32 bits mean what they say."""

from __future__ import annotations

import pytest
import torch

from tests.test_gpu_paged_attention import Batch
from tricast_b200 import paged_attention

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
@pytest.mark.parametrize("new,total", [([1, 3], [300, 90]), ([200, 1], [300, 90]), ([9], [4])])
def test_large_windows_and_bounds(dtype, new, total):
    b = Batch(new, total, 8, 2, 64, 16, "fp8_row", dtype)
    want = b.run()
    for window in ((1 << 31) - 1, 1 << 31, (1 << 32) + 5, 1 << 60):
        assert torch.equal(b.run(window=window), want), window
    for most in ((1 << 31) + 1, (1 << 32) + 1):
        got = paged_attention(b.q, b.cache, b.table, b.lens, b.cu, max_q_len=most)
        assert torch.equal(got, paged_attention(b.q, b.cache, b.table, b.lens, b.cu)), most
