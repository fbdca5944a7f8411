"""Inputs of an adapter that are infinite: the formula's infinities, not NaN."""

from __future__ import annotations

import pytest
import torch

from tricast_b200 import low_rank_add

pytestmark = pytest.mark.gpu


def inputs(tokens, k, n, rank, dtype):
    """Positive weights, so that no formula meets infinities of both signs."""
    g = torch.Generator(device="cuda").manual_seed(tokens + rank)

    def rand(*shape):
        return 0.1 + torch.rand(*shape, generator=g, device="cuda")

    index = (torch.arange(tokens, device="cuda") % 3 - 1).to(torch.int32)
    return rand(tokens, n), rand(tokens, k).to(dtype), rand(2, rank, k).to(dtype), rand(2, n, rank).to(dtype), index


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("rank", [1, 12, 16, 20, 40, 100, 128, 130])
@pytest.mark.parametrize("tokens", [3, 20, 500])
def test_an_infinite_x_gives_infinities(tokens, rank, dtype):
    """At ranks that kernels fill up to whole tiles as at others."""
    y, x, a, b, index = inputs(tokens, 72, 136, rank, dtype)
    inf = float("inf")
    x[1, 3], x[2, 70] = inf, -inf  # tokens of the adapters 0 and 1
    for out in {torch.float32, dtype}:
        got = low_rank_add(y, x, a, b, index, dtype=out)
        assert (got[1] == inf).all() and (got[2] == -inf).all()
        others = torch.ones(tokens, dtype=torch.bool, device="cuda")
        others[1:3] = False
        assert torch.isfinite(got[others]).all()


@pytest.mark.parametrize("tokens", [3, 500])
def test_beside_an_infinite_one_large_numbers_stay_finite_in_fp16(tokens):
    """h of -2e8, beyond fp16, next to an infinite one: Inf, not the difference of two."""
    y, x, a, b, index = inputs(tokens, 64, 64, 16, torch.float16)
    x[1], a[0, 0], a[0, 1, 3] = 6e4, -60.0, float("inf")
    got = low_rank_add(y, x, a, b, index)
    assert (got[1] == float("inf")).all()
