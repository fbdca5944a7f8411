"""Page plans against a plain walk over sequences and tokens."""

from __future__ import annotations

import random

import pytest
import torch

from tricast_b200 import PagedKVCache, paged_attention, plan_pages, release_pages

pytestmark = pytest.mark.gpu


def walk(lens, new, table, free, taken, page, tokens):
    """The plan token by token: the table is changed in place."""
    out, cu, slots, seq, pos, missing = [], [0], [], [], [], 0
    taken = min(max(taken, 0), len(free))
    for i, (have, want) in enumerate(zip(lens, new)):
        have = max(have, 0)
        n = min(max(want, 0), tokens - cu[-1])
        used, need = -(-have // page), -(-(have + n) // page)
        for c in range(used, need):
            if c >= len(table[i]):
                missing += 1
                continue
            if taken < len(free):
                table[i][c] = free[taken]
                taken += 1
            else:
                table[i][c] = -1
                missing += 1
        for p in range(have, have + n):
            held = table[i][p // page] if p // page < len(table[i]) else -1
            slots.append(held * page + p % page if held >= 0 else -1)
            seq.append(i)
            pos.append(p)
        out.append(have + n)
        cu.append(cu[-1] + n)
    rest = tokens - len(slots)
    return out, cu, slots + [-1] * rest, seq + [-1] * rest, pos + [-1] * rest, taken, missing


def check(lens, new, table, free, taken, page, tokens):
    as32 = dict(dtype=torch.int32, device="cuda")
    t = torch.tensor(table, **as32).view(len(lens), -1)
    f = torch.tensor(free, **as32)
    kept = f.clone()
    plan = plan_pages(torch.tensor(lens, **as32), torch.tensor(new, **as32), t, f, torch.tensor([taken], **as32),
                      page_size=page, tokens=tokens)
    want = walk(lens, new, table, free, taken, page, tokens)
    got = [plan.seq_lens, plan.cu_q, plan.slots, plan.sequence, plan.positions, plan.taken, plan.missing]
    for name, w, g in zip(plan._fields, want, [*got[:5], *got[5:]]):
        assert g.flatten().tolist() == (w if isinstance(w, list) else [w]), name
    assert t.tolist() == table and torch.equal(f, kept)
    return plan


@pytest.mark.parametrize("batch, page, most", [(1, 8, 1), (1, 16, 700), (3, 16, 40), (64, 64, 1), (257, 8, 5), (1025, 32, 3),
                                               (2500, 256, 2), (4097, 1, 2)])
def test_batches(batch, page, most):
    rng = random.Random(batch * page + most)
    lens = [rng.choice((0, 1, page - 1, page, page + 1, rng.randint(0, 5 * page))) for _ in range(batch)]
    new = [rng.choice((0, 1, most, rng.randint(0, most))) for _ in range(batch)]
    width = max(-(-(h + n) // page) for h, n in zip(lens, new)) + 2
    pages = list(range(batch * width))
    rng.shuffle(pages)
    table, at = [[-1] * width for _ in range(batch)], 0
    for i, h in enumerate(lens):
        for c in range(-(-h // page)):
            table[i][c] = pages[at]
            at += 1
    for tokens in {sum(new), sum(new) + 3}:
        check(lens, new, [list(r) for r in table], pages, at, page, tokens)


def test_what_does_not_fit():
    table = [[4, -1, -1], [-1, -1, -1], [5, 6, 7], [-1, -1, -1]]
    lens, new = [7, 0, 24, 0], [10, 9, 4, 1]

    def rows():
        return [list(r) for r in table]

    check(lens, new, rows(), [0, 1, 2, 3, 8, 9], 2, 8, 24)
    check(lens, new, rows(), [0, 1, 2, 3, 8, 9], 4, 8, 24)  # the stack runs out
    check(lens, new, rows(), [0, 1, 2, 3, 8, 9], 6, 8, 24)  # nothing is free
    check(lens, new, rows(), [], 0, 8, 24)
    check(lens, new, rows(), [0, 1, 2, 3], 9, 8, 24)  # a top beyond the stack counts as its end
    check(lens, new, rows(), [0, 1, 2, 3], -2, 8, 24)
    for tokens in (0, 1, 10, 11, 23):  # tokens beyond the room
        check(lens, new, rows(), [0, 1, 2, 3, 8, 9], 0, 8, tokens)
    check([0, -3, 5], [-1, 2, 0], [[-1], [-1], [0]], [1, 2], 0, 8, 4)  # lengths below 0 count as 0
    check([9, 20], [3, 1], [[1], [2]], [3, 4, 5], 0, 8, 4)  # sequences longer than their rows
    check([8, 3], [1, 1], [[-1, -1], [-1, -1]], [3, 4, 5], 0, 8, 2)  # pages that a row never had


def test_empty_batches():
    as32 = dict(dtype=torch.int32, device="cuda")
    none = torch.empty(0, **as32)
    plan = plan_pages(none, none, torch.empty(0, 4, **as32), none, torch.zeros(1, **as32), page_size=16, tokens=3)
    assert plan.cu_q.tolist() == [0] and plan.slots.tolist() == [-1] * 3 and plan.missing.item() == 0
    check([0, 0], [1, 2], [[], []], [1, 2], 0, 16, 3)


def test_long_sums_pass_32_bits():
    as32 = dict(dtype=torch.int32, device="cuda")
    new = torch.full((3,), (1 << 31) - 1, **as32)
    table = torch.full((3, 2), -1, **as32)
    plan = plan_pages(torch.zeros(3, **as32), new, table, torch.arange(4, **as32), torch.zeros(1, **as32), page_size=8, tokens=12)
    assert plan.cu_q.tolist() == [0, 12, 12, 12] and plan.seq_lens.tolist() == [12, 0, 0]
    assert table.tolist() == [[0, 1], [-1, -1], [-1, -1]] and plan.slots.tolist() == list(range(12))


@pytest.mark.parametrize("batch, width", [(1, 1), (5, 70), (9, 33), (300, 7), (2049, 3)])
def test_release(batch, width):
    rng = random.Random(batch + width)
    pages = list(range(batch * width + 5))
    rng.shuffle(pages)
    counts = [rng.randint(0, width) for _ in range(batch)]
    ended = [rng.random() < 0.5 for _ in range(batch)]
    free, table, at = list(pages), [], 0
    for n in counts:
        row = [-1] * width
        for c in rng.sample(range(width), n):  # holes are skipped
            row[c] = pages[at]
            at += 1
        table.append(row)
    as32 = dict(dtype=torch.int32, device="cuda")
    t, f = torch.tensor(table, **as32), torch.tensor(free, **as32)
    top = release_pages(t, torch.tensor(ended, device="cuda"), f, torch.tensor([at], **as32))
    back = [p for row, e in zip(table, ended) if e for p in row if p >= 0]
    assert top.tolist() == [at - len(back)]
    free[at - len(back):at] = back
    assert f.tolist() == free
    assert t.tolist() == [[-1] * width if e else row for row, e in zip(table, ended)]


def test_more_pages_back_than_were_taken():
    as32 = dict(dtype=torch.int32, device="cuda")
    t, f = torch.tensor([[3, 4, 5], [6, -1, -1]], **as32), torch.tensor([0, 1, 2], **as32)
    top = release_pages(t, torch.tensor([True, True], device="cuda"), f, torch.tensor([2], **as32))
    assert top.tolist() == [0] and f.tolist() == [5, 6, 2] and t.max().item() == -1


def test_rows_of_a_wider_table():
    """Strides: the rows of a slice of a table; what lies beside them stays."""
    as32 = dict(dtype=torch.int32, device="cuda")
    whole = torch.full((4, 10), -7, **as32)
    view = whole[1:3, 2:5]
    view.fill_(-1)
    plan = plan_pages(torch.zeros(2, **as32), torch.tensor([9, 17], **as32), view, torch.arange(8, **as32),
                      torch.zeros(1, **as32), page_size=8, tokens=26)
    want = torch.full((4, 10), -7, **as32)
    want[1, 2:5] = torch.tensor([0, 1, -1], **as32)
    want[2, 2:5] = torch.tensor([2, 3, 4], **as32)
    assert torch.equal(whole, want) and plan.taken.item() == 5
    release_pages(view, torch.tensor([False, True], device="cuda"), torch.arange(8, **as32), plan.taken)
    want[2, 2:5] = -1
    assert torch.equal(whole, want)


def test_a_captured_step_replays():
    """A decode loop without the host: state is copied over inside the graph."""
    as32 = dict(dtype=torch.int32, device="cuda")
    lens, new = torch.tensor([7, 0, 15], **as32), torch.tensor([1, 1, 1], **as32)
    table, free, taken = torch.full((3, 4), -1, **as32), torch.arange(12, **as32), torch.zeros(1, **as32)
    first = plan_pages(torch.zeros(3, **as32), lens, table, free, taken, page_size=8, tokens=22)
    taken.copy_(first.taken)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        plan = plan_pages(lens, new, table, free, taken, page_size=8, tokens=3)
        lens.copy_(plan.seq_lens)
        taken.copy_(plan.taken)
    rows, have, top = table.tolist(), lens.tolist(), taken.item()
    for _ in range(11):
        graph.replay()
        want = walk(have, [1, 1, 1], rows, list(range(12)), top, 8, 3)
        have, top = want[0], want[5]
        assert plan.slots.tolist() == want[2] and table.tolist() == rows and lens.tolist() == have


def test_the_cache_and_the_attention_take_a_plan():
    g = torch.Generator(device="cuda").manual_seed(1)
    as32 = dict(dtype=torch.int32, device="cuda")
    cache = PagedKVCache(20, 8, 2, 32, None)
    new = torch.tensor([5, 0, 19], **as32)
    table = torch.full((3, 5), -1, **as32)
    free = torch.randperm(20, generator=g, device="cuda").to(torch.int32)
    plan = plan_pages(torch.zeros(3, **as32), new, table, free, torch.zeros(1, **as32), page_size=8, tokens=26)
    q, k, v = (torch.randn(26, h, 32, generator=g, device="cuda").bfloat16() for h in (4, 2, 2))
    cache.write(k, v, plan.slots)
    got = paged_attention(q, cache, table, plan.seq_lens, plan.cu_q)
    for lo, hi in ((0, 5), (5, 24)):
        kk, vv = (t[lo:hi].double().repeat_interleave(2, 1) for t in (k, v))
        s = torch.einsum("qhd,khd->hqk", q[lo:hi].double(), kk) / 32 ** 0.5
        s = s.masked_fill(torch.ones_like(s[0], dtype=torch.bool).triu(1), float("-inf"))
        want = torch.einsum("hqk,khd->qhd", s.softmax(-1), vv)
        assert (got[lo:hi].double() - want).abs().max() < 0.05  # bf16 weights and outputs: 2**-8 of values up to 4, thrice
    assert got[24:].abs().max() == 0


def test_refusals():
    as32 = dict(dtype=torch.int32, device="cuda")
    i, table, top = torch.zeros(2, **as32), torch.zeros(2, 4, **as32), torch.zeros(1, **as32)

    def call(lens=i, new=i, table=table, free=i, taken=top, page=16, tokens=2):
        return plan_pages(lens, new, table, free, taken, page_size=page, tokens=tokens)

    for kw in (dict(lens=i[:1]), dict(lens=i.long()), dict(new=i.cpu()), dict(table=table.t()), dict(table=table[0]),
               dict(table=table[:1].expand(2, 4)), dict(free=table), dict(taken=i), dict(taken=top.long()), dict(page=24),
               dict(tokens=-1), dict(lens=torch.zeros(4, **as32)[::2]), dict(free=torch.zeros(4, **as32)[::2])):
        with pytest.raises(ValueError):
            call(**kw)
    with pytest.raises(ValueError, match="ended"):
        release_pages(table, i, i, top)
