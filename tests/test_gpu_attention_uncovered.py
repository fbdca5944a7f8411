"""Rows of ``q`` that no sequence covers (a batch padded to a fixed size, more new tokens than ``max_q_len``) give zeros
and -Inf, whatever the output's memory held."""

from __future__ import annotations

import pytest
import torch

from tests.test_gpu_attention_laid_out import _leave_nan_behind
from tests.test_gpu_paged_attention import Batch, _bound
from tricast_b200 import PagedKVCache, paged_attention

pytestmark = pytest.mark.gpu


def _near(b, out, lse, rows, **kw):
    want, size, want_lse = b.exact(**kw)
    assert ((out.double() - want).abs()[rows] <= _bound(b.q.dtype, b.cache.scheme) * size[rows] + 1e-30).all()
    assert ((lse.double() - want_lse)[rows].abs() <= 1e-4).all()


@pytest.mark.parametrize("scheme", [None, "fp8_row", "mxfp4"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16], ids=str)
@pytest.mark.parametrize("new,total,before,after", [([1, 1, 2], [30, 700, 9], 0, 1), ([3, 0, 1], [200, 9, 65], 2, 700),
                                                    ([150, 1, 60], [300, 20, 90], 5, 333), ([300], [900], 1, 0)])
def test_padding_before_and_after(scheme, dtype, new, total, before, after):
    b = Batch(new, total, 8, 2, 64, 16, scheme, dtype, seed=after)
    n = sum(new)
    junk = torch.full((before + n + after, 8, 64), float("nan"), dtype=dtype, device="cuda")
    junk[before:before + n] = b.q
    _leave_nan_behind()
    out, lse = paged_attention(junk, b.cache, b.table, b.lens, b.cu + before, max_q_len=max(new), return_lse=True)
    rest = torch.ones(before + n + after, dtype=torch.bool, device="cuda")
    rest[before:before + n] = False
    assert (out[rest] == 0).all() and (lse[rest] == float("-inf")).all()
    _near(b, out[~rest], lse[~rest], slice(None))


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
@pytest.mark.parametrize("new,total,most", [([5, 1, 9], [40, 3, 9], 3), ([5, 1, 9], [40, 300, 9], 1), ([400, 1, 90], [900, 33, 90], 150)])
def test_more_tokens_than_max_q_len(causal, dtype, new, total, most):
    """The first ``max_q_len`` of them keep their positions; the others are not computed."""
    b = Batch(new, total, 8, 2, 64, 16, "fp8_row", dtype, seed=most)
    _leave_nan_behind()
    out, lse = paged_attention(b.q, b.cache, b.table, b.lens, b.cu, max_q_len=most, return_lse=True, causal=causal)
    kept = torch.cat([torch.arange(n) < most for n in new]).cuda()
    assert (out[~kept] == 0).all() and (lse[~kept] == float("-inf")).all()
    _near(b, out, lse, kept, causal=causal)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16], ids=str)
def test_no_sequences(dtype):
    cache = PagedKVCache(2, 16, 2, 64, dtype=dtype)
    empty = torch.empty(0, dtype=torch.int32, device="cuda")
    q = torch.randn(70, 4, 64, device="cuda").to(dtype)
    _leave_nan_behind()
    out, lse = paged_attention(q, cache, empty.view(0, 3), empty, torch.zeros(1, dtype=torch.int32, device="cuda"),
                               return_lse=True)
    assert (out == 0).all() and (lse == float("-inf")).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
@pytest.mark.parametrize("new", [[1, 1], [200, 3]])
def test_a_table_without_pages(dtype, new):
    """No sequence has a page: none of its tokens sees a key."""
    cache = PagedKVCache(2, 16, 2, 64, dtype=dtype)
    q = torch.randn(sum(new), 8, 64, device="cuda").to(dtype)
    cu = torch.tensor([0, new[0], sum(new)], dtype=torch.int32, device="cuda")
    _leave_nan_behind()
    for lens in ([0, 0], [5, 900]):
        out, lse = paged_attention(q, cache, torch.empty((2, 0), dtype=torch.int32, device="cuda"),
                                   torch.tensor(lens, dtype=torch.int32, device="cuda"), cu, max_q_len=max(new), return_lse=True)
        assert (out == 0).all() and (lse == float("-inf")).all()


def test_a_padded_batch_in_a_graph():
    """The same graph with other counts of tokens: what is padding is read on the device."""
    b = Batch([6, 1, 4], [90, 300, 64], 8, 2, 128, 16, "fp8_row", torch.bfloat16)
    q = torch.zeros(16, 8, 128, dtype=torch.bfloat16, device="cuda")
    q[:11] = b.q
    paged_attention(q, b.cache, b.table, b.lens, b.cu, max_q_len=6)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, lse = paged_attention(q, b.cache, b.table, b.lens, b.cu, max_q_len=6, return_lse=True)
    for cu in ([0, 6, 7, 11], [2, 5, 5, 9], [0, 0, 1, 1]):
        b.cu.copy_(torch.tensor(cu, dtype=torch.int32))
        out.fill_(float("nan"))
        lse.fill_(float("nan"))
        graph.replay()
        rest = torch.ones(16, dtype=torch.bool, device="cuda")
        rest[cu[0]:cu[-1]] = False
        assert (out[rest] == 0).all() and (lse[rest] == float("-inf")).all()
        again, _ = paged_attention(q, b.cache, b.table, b.lens, b.cu, max_q_len=6, return_lse=True)
        assert torch.equal(out, again) and torch.isfinite(out).all()
