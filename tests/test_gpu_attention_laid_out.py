"""Chunks of so many query rows that the quantized operands are laid out once, before the attention kernel: the
same checks, with the same tolerances (``test_gpu_paged_attention``), at the places where the layout can go wrong."""

from __future__ import annotations

import pytest
import torch

from tests.test_gpu_paged_attention import Batch, _bound
from tricast_b200 import _native as N
from tricast_b200 import paged_attention

pytestmark = pytest.mark.gpu

SCHEMES = ["fp8_row", "int8_row", "mxfp4"]


def _leave_nan_behind(nbytes=1 << 28):
    """What the allocator hands out next has been NaN in every type."""
    junk = torch.full((nbytes,), 0xFF, dtype=torch.uint8, device="cuda")
    del junk


@pytest.mark.parametrize("scheme", SCHEMES)
@pytest.mark.parametrize("heads,kv_heads,dim,page,dtype", [(8, 1, 128, 64, torch.bfloat16), (12, 2, 64, 8, torch.float16),
                                                           (16, 2, 96, 16, torch.bfloat16), (8, 1, 32, 256, torch.float16)])
def test_heads_pages_and_lengths(scheme, heads, kv_heads, dim, page, dtype):
    _leave_nan_behind()
    Batch([130, 1, 0, 5, 200], [130, 257, 40, 5, 900], heads, kv_heads, dim, page, scheme, dtype, seed=page).check()


@pytest.mark.parametrize("scheme", SCHEMES)
@pytest.mark.parametrize("window", [1, 127, 128, 129, 400])
def test_windows_skip_what_no_row_sees(scheme, window):
    _leave_nan_behind()
    Batch([200, 1, 33], [1500, 700, 1025], 8, 1, 128, 16, scheme, torch.bfloat16, seed=window).check(window=window)


@pytest.mark.parametrize("scheme", SCHEMES)
def test_rows_and_sequences_without_keys(scheme):
    _leave_nan_behind()
    Batch([200, 100, 150, 3], [90, 0, 150, 1], 8, 1, 64, 16, scheme, torch.bfloat16).check()


@pytest.mark.parametrize("scheme", SCHEMES)
def test_absent_pages(scheme):
    _leave_nan_behind()
    b = Batch([160], [640], 8, 1, 128, 16, scheme, torch.bfloat16)
    full = b.run()
    b.table[0, 1] = b.cache.num_pages + 5
    b.table[0, 7:9] = -1
    gone = torch.zeros(640, dtype=torch.bool, device="cuda")
    gone[16:32] = gone[112:144] = True
    out, lse = b.run(return_lse=True)
    q, k, v = b.q.double(), b.k[0], b.v[0]
    seen = torch.arange(640, device="cuda")[None] <= torch.arange(480, 640, device="cuda")[:, None]
    s = torch.einsum("ihd,jd->hij", q, k[:, 0]) / 128 ** 0.5
    p = torch.softmax(s.masked_fill(~(seen & ~gone)[None], float("-inf")), -1)
    want, size = torch.einsum("hij,jd->ihd", p, v[:, 0]), torch.einsum("hij,jd->ihd", p, v[:, 0].abs())
    assert ((out.double() - want).abs() <= _bound(torch.bfloat16, scheme) * size).all()
    assert not torch.equal(full, out)


def test_scales_that_are_not_numbers_reach_only_the_rows_that_see_them():
    b = Batch([200], [500], 8, 1, 64, 16, "fp8_row", torch.bfloat16)
    clean = b.run()
    page, at = int(b.table[0, 450 // 16]), 450 % 16
    b.cache.v_scale[page, 0, at] = float("nan")
    out = b.run()
    assert torch.equal(out[:150], clean[:150])  # token i sits at position 300 + i
    assert torch.isnan(out[150:]).all()


def test_a_table_too_wide_for_the_layout_gives_the_same_result():
    b = Batch([200, 60], [900, 700], 16, 2, 128, 16, "fp8_row", torch.bfloat16)
    wide = torch.full((2, 1 << 15), -1, dtype=torch.int32, device="cuda")  # 2**19 positions a sequence
    wide[:, : b.table.shape[1]] = b.table
    lib = N.lib()

    def room(pages):
        return lib.tc_paged_attention_workspace(b.cache._ref, 16, 260, 2, 200, pages)

    assert room(wide.shape[1]) < room(b.table.shape[1])
    b.check()
    b.table = wide
    b.check()


@pytest.mark.parametrize("polls", [0, 1, 20])
def test_waits_that_run_out(polls):
    b = Batch([150, 1, 300], [300, 40, 800], 8, 1, 128, 16, "fp8_row", torch.bfloat16)
    N.lib().tc_set_wait_limit(polls)
    try:
        b.check()
    finally:
        N.lib().tc_set_wait_limit(-1)


def test_streams_and_graphs():
    b = Batch([256, 100], [1000, 900], 8, 1, 128, 64, "mxfp4", torch.bfloat16)
    want = b.run()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = b.run()
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = paged_attention(b.q, b.cache, b.table, b.lens, b.cu, max_q_len=256)
    b.q.mul_(0.5)
    want = b.run()
    graph.replay()
    assert torch.equal(got, want)
