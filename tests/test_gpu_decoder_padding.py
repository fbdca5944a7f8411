"""Batches with room behind their last token: what stands there changes nothing."""

from __future__ import annotations

import pytest
import torch

from tricast_b200 import PagedKVCache, plan_pages
from tricast_b200.serving import random_decoder


@pytest.mark.gpu
@pytest.mark.parametrize("scheme", [None, "fp8_row"])
def test_padding_ids_change_no_logit(scheme):
    decoder = random_decoder(vocab=300, hidden=64, heads=2, kv_heads=1, inner=96, adapters=2, seed=6)
    as32 = dict(dtype=torch.int32, device="cuda")
    ids, new = [5, 299, 0, 17, 3], torch.tensor([3, 0, 2], **as32)

    def logits(padding):
        caches = [PagedKVCache(4, 8, a.kv_heads, a.head_dim, scheme, dtype=a.dtype) for a, _ in decoder.layers]
        table, zero = torch.full((3, 2), -1, **as32), torch.zeros(3, **as32)
        plan = plan_pages(zero, new, table, torch.arange(4, **as32), torch.zeros(1, **as32), page_size=8, tokens=9)
        index = torch.tensor([0, 0, 0, 1, 1, -1, 0, 1, 7], **as32)
        out = decoder(torch.tensor(ids + padding, device="cuda"), caches, plan, table, max_q_len=3, index=index)
        return out[[0, 2]]  # the second sequence has no new token

    want = logits([0, 0, 0, 0])
    assert torch.isfinite(want).all()
    for padding in ([1, 2, 3, 4], [299, 0, 299, 0], [-1, 300, -(2 ** 62), 2 ** 62]):
        assert torch.equal(logits(padding), want)
