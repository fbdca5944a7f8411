"""The attention layer called as its documentation shows, without a bound on the new tokens."""

from __future__ import annotations

import pytest
import torch

from tests.test_gpu_attention_laid_out import _leave_nan_behind
from tricast_b200 import PagedKVCache
from tricast_b200.serving import AttentionLayer

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("lens", [[9], [40, 3], [1, 1, 1]])
def test_the_bound_may_be_left_out(lens):
    g = torch.Generator(device="cuda").manual_seed(3)

    def randn(*shape):
        return (torch.randn(*shape, generator=g, device="cuda") * 0.2).bfloat16()

    layer = AttentionLayer(randn((4 + 2 * 2) * 32, 128), randn(128, 4 * 32), randn(128), 4, 2)
    total, page = sum(lens), 16
    pages = [-(-n // page) for n in lens]
    table = torch.full((len(lens), max(pages)), -1, dtype=torch.int32)
    at = 0
    slots = []
    for i, n in enumerate(lens):
        table[i, : pages[i]] = torch.arange(at, at + pages[i])
        slots.append(at * page + torch.arange(n))
        at += pages[i]
    x, r, table, slots = randn(total, 128), randn(total, 128), table.cuda(), torch.cat(slots).cuda()
    context = torch.tensor(lens, dtype=torch.int32, device="cuda")
    cu = torch.nn.functional.pad(context.cumsum(0), (1, 0)).to(torch.int32)
    want, h = layer(x, r, PagedKVCache(at, page, 2, 32), slots, table, context, cu, max_q_len=max(lens))
    _leave_nan_behind()
    got, same = layer(x, r, PagedKVCache(at, page, 2, 32), slots, table, context, cu)
    assert torch.equal(got, want) and torch.equal(same, h)
