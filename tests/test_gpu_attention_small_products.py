"""Attention where a score's factors vanish: a scale of the scores of 0 or next to it with small queries. Hidden keys stay
hidden and the rest has its weight."""

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
