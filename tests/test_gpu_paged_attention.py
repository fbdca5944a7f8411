"""Attention over the quantized paged cache against the formula in 64 bits on the cache's own values.

Tolerance, by the arithmetic (``_bound``, in units of sum_j p_j |v_j|): a weight is rounded once to the 16-bit
type of its product with the values (fp16 over quantized caches, the cache's own type otherwise) and the
result once to its type; rounding to nearest is off by at most 2**-8 of a bf16 value (8 significant bits) and
2**-11 of an fp16 value. fp32 scores, exponentials and sums add less than 1e-4. In fp32 nothing is rounded below
32 bits: scores of magnitude up to 100 carry 1e-5, so 4e-5."""

from __future__ import annotations

import itertools
import math

import pytest
import torch

from tricast_b200 import PagedKVCache, paged_attention
from tricast_b200 import _native as N

pytestmark = pytest.mark.gpu

SCHEMES = [None, "fp8_row", "int8_row", "mxfp4"]


UNIT = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def _bound(dtype, scheme):
    if dtype == torch.float32:
        return 4e-5
    return UNIT[dtype if scheme is None else torch.float16] + UNIT[dtype] + 1e-4


class Batch:
    """Sequences with shuffled pages; whatever lies past a context in its last page is not finite."""

    def __init__(self, new, total, heads, kv_heads, dim, page, scheme, dtype, seed=0, q_scale=1.5):
        g = torch.Generator().manual_seed(seed)
        self.new, self.total, self.heads, self.kv_heads, self.dim = new, total, heads, kv_heads, dim
        need = [max(0, -(-t // page)) for t in total]
        pages = sum(need) + 2
        self.cache = PagedKVCache(pages, page, kv_heads, dim, scheme, dtype=dtype)
        order = torch.randperm(pages, generator=g)
        self.table = torch.full((len(total), max(max(need), 1)), -1, dtype=torch.int32)
        self.k, self.v = [], []
        at = 0
        everything = torch.full((pages * page, kv_heads, dim), float("inf"), dtype=dtype).cuda()
        self.cache.write(everything, everything, torch.arange(pages * page).cuda())
        for b, (n, t) in enumerate(zip(need, total)):
            mine = order[at:at + n]
            at += n
            self.table[b, :n] = mine.int()
            pos = torch.arange(max(t, 0))
            slots = (mine[pos // page] * page + pos % page).cuda()
            k = torch.randn(len(pos), kv_heads, dim, generator=g) * 0.5
            k[..., torch.randperm(dim, generator=g)[: max(1, dim // 64)]] *= 8
            v = torch.randn(len(pos), kv_heads, dim, generator=g)
            self.cache.write(k.to(dtype).cuda(), v.to(dtype).cuda(), slots)
            self.k.append(self._values(self.cache.k, self.cache.k_scale, slots, page))
            self.v.append(self._values(self.cache.v, self.cache.v_scale, slots, page))
        self.q = (torch.randn(sum(new), heads, dim, generator=g) * q_scale).to(dtype).cuda()
        self.lens = torch.tensor(total, dtype=torch.int32).cuda()
        self.cu = torch.tensor([0, *itertools.accumulate(new)], dtype=torch.int32).cuda()
        self.table = self.table.cuda()

    def _values(self, pool, scales, slots, page):
        p, o = slots // page, slots % page
        if self.cache.scheme is None:
            return pool[p, :, o].double()
        c = pool.view(torch.uint8)[p, :, o]
        if self.cache.scheme == "mxfp4":
            grid = torch.tensor([0, .5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64, device="cuda")
            grid = torch.cat([grid, -grid])
            v = grid[torch.stack([c & 15, c >> 4], -1).flatten(-2).long()]
            s = torch.pow(2.0, scales.view(torch.uint8)[p, :, o].double() - 127)
            return v * s.repeat_interleave(32, -1)
        return c.view(pool.dtype).double() * scales[p, :, o].double()[..., None]

    def run(self, **kw):
        return paged_attention(self.q, self.cache, self.table, self.lens, self.cu, max_q_len=max(max(self.new), 1), **kw)

    def exact(self, scale=None, causal=True, window=0):
        scale = 1 / math.sqrt(self.dim) if scale is None else scale
        outs, sizes, lses = [], [], []
        at = 0
        group = self.heads // self.kv_heads
        for n, t, k, v in zip(self.new, self.total, self.k, self.v):
            q = self.q[at:at + n].double()
            at += n
            pos = torch.arange(max(t, 0), device="cuda")
            here = torch.arange(n, device="cuda") + (t - n)
            seen = torch.ones(n, len(pos), dtype=torch.bool, device="cuda")
            if causal:
                seen = pos[None] <= here[:, None]
                if window:
                    seen &= pos[None] > here[:, None] - window
            kk, vv = k.repeat_interleave(group, 1), v.repeat_interleave(group, 1)
            s = torch.einsum("ihd,jhd->hij", q, kk) * scale
            s = s.masked_fill(~seen[None], float("-inf"))
            lse = torch.logsumexp(s, -1)
            p = torch.where(lse[..., None] == float("-inf"), 0.0, torch.exp(s - torch.where(lse == float("-inf"), 0.0, lse)[..., None]))
            outs.append(torch.einsum("hij,jhd->ihd", p, vv))
            sizes.append(torch.einsum("hij,jhd->ihd", p, vv.abs()))
            lses.append(lse.T)
        return torch.cat(outs), torch.cat(sizes), torch.cat(lses)

    def check(self, **kw):
        out, lse = self.run(return_lse=True, **kw)
        want, size, want_lse = self.exact(**kw)
        tol = _bound(self.q.dtype, self.cache.scheme)
        assert out.dtype == self.q.dtype and out.shape == self.q.shape
        assert torch.isfinite(out).all()
        assert ((out.double() - want).abs() <= tol * size + 1e-30).all(), ((out.double() - want).abs() / (size + 1e-30)).max()
        empty = want_lse == float("-inf")
        assert torch.equal(lse == float("-inf"), empty)
        assert (out[empty] == 0).all()
        assert ((lse.double() - want_lse)[~empty].abs() <= 1e-4).all()
        only = self.run(**kw)
        assert torch.equal(only, out)


@pytest.mark.parametrize("scheme", SCHEMES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16], ids=str)
@pytest.mark.parametrize("heads,kv_heads,dim,page", [(4, 4, 64, 16), (8, 1, 128, 64), (12, 4, 128, 8), (5, 1, 32, 32),
                                                     (6, 2, 96, 16), (4, 2, 256, 32), (16, 1, 160, 128), (20, 1, 64, 256)])
def test_types_and_heads(scheme, dtype, heads, kv_heads, dim, page):
    Batch([1, 3, 0, 17, 40], [77, 3, 9, 130, 1000], heads, kv_heads, dim, page, scheme, dtype, seed=dim).check()


@pytest.mark.parametrize("scheme", SCHEMES)
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("total", [1, 2, 15, 16, 17, 63, 64, 65, 127, 128, 129, 255, 257, 511, 1023, 4097])
def test_one_token_at_every_edge(scheme, dim, total):
    Batch([1, 1], [total, max(1, total // 2)], 8, 2, dim, 16, scheme, torch.bfloat16, seed=total).check()


@pytest.mark.parametrize("scheme", SCHEMES)
@pytest.mark.parametrize("new,total", [(2, 2), (7, 7), (16, 300), (31, 32), (64, 64), (65, 1000), (127, 128), (128, 128),
                                       (129, 129), (200, 201), (256, 1300), (257, 600), (513, 513), (1000, 1001)])
def test_chunks(scheme, new, total):
    for dim, dtype, page in ((128, torch.bfloat16, 64), (64, torch.float16, 16)):
        Batch([new], [total], 8, 2, dim, page, scheme, dtype, seed=new).check()


@pytest.mark.parametrize("scheme", SCHEMES)
@pytest.mark.parametrize("window", [1, 2, 63, 64, 100, 128, 1000, 5000])
def test_windows(scheme, window):
    for dim, new in ((128, [1, 1, 4]), (64, [1, 200, 333])):
        Batch(new, [1500, 200, 700], 6, 2, dim, 32, scheme, torch.bfloat16, seed=window).check(window=window)


@pytest.mark.parametrize("scheme", [None, "fp8_row"])
def test_not_causal_and_scale(scheme):
    for new in ([1, 5, 2], [300, 4, 150]):
        b = Batch(new, [500, 129, 400], 8, 4, 128, 16, scheme, torch.bfloat16)
        b.check(causal=False)
        b.check(causal=False, scale=0.02)
        b.check(scale=0.0)
        b.check(scale=-0.05)


@pytest.mark.parametrize("scheme", SCHEMES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
def test_rows_that_see_nothing(scheme, dtype):
    """More new tokens than context (their positions lie before the first key), and empty contexts."""
    for new, total in (([3, 1, 2], [1, 0, 0]), ([200, 150, 1], [40, 0, 0]), ([1, 1], [0, 0])):
        Batch(new, total, 4, 2, 64, 16, scheme, dtype).check()


@pytest.mark.parametrize("scheme", [None, "fp8_row", "mxfp4"])
def test_many_heads_per_key_head_and_long_context(scheme):
    Batch([1], [30000], 32, 1, 128, 64, scheme, torch.bfloat16).check()
    Batch([3, 1], [20011, 5], 40, 1, 128, 64, scheme, torch.bfloat16).check()
    Batch([2, 130], [9000, 8001], 16, 2, 64, 128, scheme, torch.float16).check()


@pytest.mark.parametrize("scheme", [None, "int8_row"])
def test_large_and_extreme_scores(scheme):
    """Scores in the hundreds, so that the running maximum moves and single keys take all the weight; and
    scores that differ by more than fp32's exponent range."""
    for new in ([1, 1], [140, 300]):
        b = Batch(new, [700, 900], 8, 2, 64, 16, scheme, torch.bfloat16, q_scale=1.5)
        out = b.run(scale=20.0)
        want, size, lse = b.exact(scale=20.0)
        # A score of magnitude s carries s * 64 * 2**-24 of error into its weight.
        top = lse.abs().max().item()
        tol = _bound(torch.bfloat16, scheme) + 4 * top * 64 * 2.0 ** -24
        assert torch.isfinite(out).all()
        assert ((out.double() - want).abs() <= tol * (size + b.v[0].abs().max())).all()


@pytest.mark.parametrize("scheme", SCHEMES)
def test_absent_pages_count_as_masked(scheme):
    """A page entry outside the cache hides its keys, as if they were not there."""
    for new in ([1], [130]):
        b = Batch(new, [640], 4, 2, 64, 16, scheme, torch.bfloat16)
        out, lse = b.run(return_lse=True, causal=False)
        b.table[0, 3] = -1
        b.table[0, 10] = b.cache.num_pages
        b.table[0, 39] = 1 << 30
        gone = torch.ones(640, dtype=torch.bool, device="cuda")
        for p in (3, 10, 39):
            gone[16 * p:16 * p + 16] = False
        got, _ = b.run(return_lse=True, causal=False)
        b.k[0], b.v[0], b.total[0] = b.k[0][gone], b.v[0][gone], int(gone.sum())
        want, size, _ = b.exact(causal=False)
        assert ((got.double() - want).abs() <= _bound(torch.bfloat16, scheme) * size).all()
        assert not torch.equal(got, out)


def test_every_page_absent():
    for new in ([1], [130]):
        b = Batch(new, [300], 4, 2, 64, 16, "fp8_row", torch.bfloat16)
        b.table.fill_(-1)
        out, lse = b.run(return_lse=True)
        assert (out == 0).all() and (lse == float("-inf")).all()


def test_strides_streams_and_repetition():
    b = Batch([1, 70, 260], [600, 500, 700], 8, 2, 128, 16, "fp8_row", torch.bfloat16)
    out = b.run()
    wide = torch.full((b.q.shape[0], 20, 131), float("nan"), dtype=torch.bfloat16, device="cuda")
    wide[:, 3:11, 1:129] = b.q
    plain = b.q
    for view in (wide[:, 3:11, 1:129], plain.transpose(0, 1).contiguous().transpose(0, 1)):
        b.q = view
        assert torch.equal(b.run(), out)
    table = torch.full((3, 2 * b.table.shape[1] + 1), -7, dtype=torch.int32, device="cuda")
    table[:, 1:1 + b.table.shape[1]] = b.table
    b.table = table[:, 1:1 + b.table.shape[1]]
    assert torch.equal(b.run(), out)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = [b.run() for _ in range(3)]
    main = b.run()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, out) for a in (*again, main))


def test_a_call_without_cu_q_and_in_a_graph():
    b = Batch([1] * 5, [5, 900, 77, 1, 2000], 8, 2, 128, 64, "fp8_row", torch.bfloat16)
    want = b.run()
    assert torch.equal(paged_attention(b.q, b.cache, b.table, b.lens), want)
    graph = torch.cuda.CUDAGraph()
    paged_attention(b.q, b.cache, b.table, b.lens)
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        out = paged_attention(b.q, b.cache, b.table, b.lens)
    # Lengths are read on the device: the graph serves other contexts than those it was captured with.
    b.lens -= torch.tensor([2, 300, 0, 0, 1999], dtype=torch.int32, device="cuda")
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, paged_attention(b.q, b.cache, b.table, b.lens))
    b.total = b.lens.tolist()
    b.k, b.v = [k[:t] for k, t in zip(b.k, b.total)], [v[:t] for v, t in zip(b.v, b.total)]
    exact, size, _ = b.exact()
    assert ((out.double() - exact).abs() <= _bound(torch.bfloat16, "fp8_row") * size).all()


def test_pool_offsets_beyond_32_bits():
    """Pages at the far end of a pool of more than 2**32 bytes."""
    pages, page = 70000, 64
    cache = PagedKVCache(pages, page, 8, 128, "fp8_row")
    g = torch.Generator().manual_seed(9)
    k, v = (torch.randn(300, 8, 128, generator=g).bfloat16().cuda() for _ in range(2))
    low = torch.arange(5, dtype=torch.int32)
    for new in (1, 300):
        outs = []
        for first in (0, pages - 5):
            table = (low + first)[None].cuda()
            cache.write(k, v, torch.arange(first * page, first * page + 300).cuda())
            q = torch.randn(new, 16, 128, generator=torch.Generator().manual_seed(1)).bfloat16().cuda()
            outs.append(paged_attention(q, cache, table, torch.tensor([300], dtype=torch.int32).cuda(),
                                        torch.tensor([0, new], dtype=torch.int32).cuda(), max_q_len=new))
        assert torch.equal(*outs)


def test_lengths_beyond_the_table_are_clamped():
    b = Batch([1, 130], [64, 640], 4, 2, 64, 16, "fp8_row", torch.bfloat16)
    want = b.run()
    b.table = b.table[:, :40].contiguous()
    b.lens[1] = 1 << 30
    assert torch.equal(b.run()[1:], want[1:])


@pytest.mark.parametrize("polls", [0, 1])
@pytest.mark.parametrize("scheme", SCHEMES)
def test_a_wait_that_runs_out_still_gives_the_result(scheme, polls):
    """With the pipeline waits limited to none or one poll the chunk kernel gives up; what runs after it
    computes the call again."""
    b = Batch([130, 1, 300], [300, 40, 300], 4, 2, 128, 16, scheme, torch.bfloat16)
    N.lib().tc_set_wait_limit(polls)
    try:
        b.check()
    finally:
        N.lib().tc_set_wait_limit(-1)
    b.check()


def test_no_tokens_and_refusals():
    b = Batch([2, 1], [40, 50], 4, 2, 64, 16, "fp8_row", torch.bfloat16)
    none = paged_attention(b.q[:0], b.cache, b.table, b.lens, torch.zeros_like(b.cu))
    assert none.shape == (0, 4, 64)
    for args in ((b.q.half(), b.cache, b.table, b.lens, b.cu), (b.q[..., :32], b.cache, b.table, b.lens, b.cu),
                 (b.q[:, :3], b.cache, b.table, b.lens, b.cu), (b.q.cpu(), b.cache, b.table, b.lens, b.cu),
                 (b.q, b.cache, b.table.long(), b.lens, b.cu), (b.q, b.cache, b.table, b.lens[:1], b.cu),
                 (b.q, b.cache, b.table, b.lens.long(), b.cu), (b.q, b.cache, b.table, b.lens, b.cu[:2]),
                 (b.q, b.cache, b.table, b.lens), (b.q, b.cache, b.table[0], b.lens, b.cu)):
        with pytest.raises(ValueError):
            paged_attention(*args)
    for kw in (dict(window=-1), dict(window=3, causal=False), dict(max_q_len=0), dict(scale=float("nan"))):
        with pytest.raises(ValueError):
            paged_attention(b.q, b.cache, b.table, b.lens, b.cu, **kw)
