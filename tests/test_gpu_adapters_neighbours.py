"""A token's bits do not depend on the other tokens of its batch."""

from __future__ import annotations

import pytest
import torch

from tricast_b200 import low_rank_add
from tricast_b200.operand import QTensor
from tricast_b200.spec import get_scheme

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype, y_dtype, out_dtype, codes", [
    (torch.bfloat16, torch.float32, torch.bfloat16, False), (torch.bfloat16, torch.bfloat16, torch.bfloat16, False),
    (torch.bfloat16, torch.float32, torch.float32, False), (torch.float16, torch.float32, torch.float16, False),
    (torch.bfloat16, torch.float32, torch.bfloat16, True), (torch.float32, torch.float32, torch.float32, False)])
@pytest.mark.parametrize("k, n", [(1032, 264), (333, 77)])
@pytest.mark.parametrize("rank", [16, 32, 64, 128])
@pytest.mark.parametrize("tokens", [2, 7, 64, 250, 700])
def test_other_tokens_change_no_bit(tokens, rank, k, n, dtype, y_dtype, out_dtype, codes):
    """The same tokens among neighbours with their adapter, each with one of their own, without any, and in another order."""
    g = torch.Generator(device="cuda").manual_seed(tokens + rank)

    def randn(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    adapters = 40
    y, x, scale = randn(tokens, n).to(y_dtype), randn(tokens, k).to(dtype), 0.5 + randn(tokens, 1).abs()
    if codes:
        x = (x.float() * 20).to(torch.float8_e4m3fn)
    a, b, gain = randn(adapters, rank, k).to(dtype), randn(adapters, n, rank).to(dtype), randn(adapters)
    t = torch.arange(tokens, device="cuda")
    index = (t // 9 % 5).to(torch.int32)

    def run(y, x, scale, index):
        if codes:
            x = QTensor(x, scale, None, None, get_scheme("fp8_row"), tuple(x.shape))
        return low_rank_add(y, x, a, b, index, gain=gain, dtype=out_dtype)

    want = run(y, x, scale, index)
    keep = t % 3 == 1
    for others in (index[keep][0].expand(tokens), (5 + t % (adapters - 5)).to(torch.int32), torch.full_like(index, -1), index.flip(0)):
        got = run(y, x, scale, torch.where(keep, index, others))
        assert torch.equal(got[keep], want[keep])
    noise = randn(tokens, k).to(x.dtype) if not codes else x.flip(0)
    got = run(torch.where(keep[:, None], y, y.flip(0)), torch.where(keep[:, None], x.float(), noise.float()).to(x.dtype),
              torch.where(keep[:, None], scale, 2 * scale), index)
    assert torch.equal(got[keep], want[keep])
    order = torch.randperm(tokens, generator=g, device="cuda")
    got = run(y[order], x.view(torch.uint8)[order].view(x.dtype) if codes else x[order], scale[order].contiguous(), index[order].contiguous())
    assert torch.equal(got, want[order])
