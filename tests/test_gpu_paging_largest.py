"""Page plans at the ends of their numbers."""

from __future__ import annotations

import pytest
import torch

from tricast_b200 import plan_pages

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("batch", [4, 1500])
def test_lengths_stay_in_32_bits(batch):
    """Tokens that would make a sequence longer than 2**31 - 1 are left out, its neighbours' come as they are."""
    as32 = dict(dtype=torch.int32, device="cuda")
    most = 2 ** 31 - 1
    lens, new = torch.zeros(batch, **as32), torch.zeros(batch, **as32)
    lens[:4], new[:4] = torch.tensor([most - 2, 0, most, 8], **as32), torch.tensor([5, 3, most, 2], **as32)
    table = torch.full((batch, 2), -1, **as32)
    table[3, 0] = 9
    plan = plan_pages(lens, new, table, torch.arange(5, **as32), torch.zeros(1, **as32), page_size=8, tokens=10)
    assert plan.seq_lens[:4].tolist() == [most, 3, most, 10] and plan.cu_q[:5].tolist() == [0, 2, 5, 5, 7]
    assert plan.sequence.tolist() == [0, 0, 1, 1, 1, 3, 3, -1, -1, -1]
    assert plan.positions.tolist() == [most - 2, most - 1, 0, 1, 2, 8, 9, -1, -1, -1]
    assert plan.slots.tolist() == [-1, -1, 0, 1, 2, 8, 9, -1, -1, -1]  # the first is longer than its row
    assert table[:4].tolist() == [[-1, -1], [0, -1], [-1, -1], [9, 1]] and plan.taken.item() == 2


@pytest.mark.parametrize("page_size", [2 ** 32 + 16, 2 ** 21, -(2 ** 32) + 16, 0, -16])
def test_page_sizes_that_are_none(page_size):
    one = torch.ones(1, dtype=torch.int32, device="cuda")
    table = torch.full((1, 4), -1, dtype=torch.int32, device="cuda")
    with pytest.raises(ValueError, match="page_size"):
        plan_pages(one * 0, one, table, one, one * 0, page_size=page_size, tokens=1)
    assert (table == -1).all()
