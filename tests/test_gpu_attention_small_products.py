"""Attention where a score's factors vanish: scales of 0 in slots that were never written, a scale of the scores of 0
or next to it with small queries. Hidden keys stay hidden and the rest has its weight."""

from __future__ import annotations

import pytest
import torch

from tests.test_gpu_paged_attention import Batch

pytestmark = pytest.mark.gpu

SHAPES = [(1, 300, 8, 2), (4, 300, 8, 2), (150, 500, 8, 2), (200, 500, 8, 1)]


@pytest.mark.parametrize("scheme", ["fp8_row", "int8_row", "mxfp4"])
@pytest.mark.parametrize("new,total,heads,kv_heads", SHAPES)
@pytest.mark.parametrize("scale,q_scale", [(0.0, 1e-5), (0.0, 1e-30), (1e-30, 1e-20), (-1e-30, 1e-20)])
def test_scores_that_vanish(scheme, new, total, heads, kv_heads, scale, q_scale):
    Batch([new], [total], heads, kv_heads, 64, 16, scheme, torch.bfloat16, seed=new, q_scale=q_scale).check(scale=scale)


@pytest.mark.parametrize("scheme", ["fp8_row", "int8_row"])
@pytest.mark.parametrize("new,total,heads,kv_heads", SHAPES)
def test_slots_that_were_never_written(scheme, new, total, heads, kv_heads):
    """Codes and scales of 0, inside the context: keys of 0 whose values are 0, for the rows that see them."""
    b = Batch([new], [total], heads, kv_heads, 64, 16, scheme, torch.bfloat16, seed=new)
    for pos in (total - 1, total - 2, 3):
        page, at = int(b.table[0, pos // 16]), pos % 16
        for pool, scales, values in ((b.cache.k, b.cache.k_scale, b.k[0]), (b.cache.v, b.cache.v_scale, b.v[0])):
            pool.view(torch.uint8)[page, :, at] = 0
            scales[page, :, at] = 0
            values[pos] = 0
    b.check()
    b.check(window=50)
