"""Attention where the values' scales differ widely or are not finite: a key that a row does not see leaves the row
alone, whatever its values are, and one that it sees acts on the elements that its values reach.

The reference is the formula in 64 bits on the cache's own values, the tolerance that of ``test_gpu_paged_attention``
(in units of sum_j p_j |v_j| over what is finite)."""

from __future__ import annotations

import math

import pytest
import torch

from tests.test_gpu_paged_attention import Batch, _bound

pytestmark = pytest.mark.gpu

# (new tokens, context, heads, key heads, window): one token, drafted tokens, a chunk whose operands every row tile
# converts, one whose operands are laid out once, and both with a window that ends inside a unit of keys.
SHAPES = [(1, 300, 8, 2, 100), (4, 300, 8, 2, 0), (150, 500, 8, 2, 0), (200, 500, 8, 1, 0), (150, 700, 8, 2, 70), (200, 700, 8, 1, 70)]


def _held(b, pool, scales, slots, page):
    """What a slot stands for: code times scale in fp32, an E8M0 scale of 255 not a number."""
    x = b._values(pool, scales, slots, page).float().double()
    if b.cache.scheme == "mxfp4":
        nan = scales.view(torch.uint8)[slots // page, :, slots % page] == 255
        x = torch.where(nan.repeat_interleave(32, -1), float("nan"), x)
    return x


def _put(b, pos, k=None, v=None):
    """Writes keys or values of the only sequence's tokens at ``pos`` again."""
    page = b.cache.page_size
    at = torch.as_tensor(pos)
    slots = (b.table[0].cpu().long()[at // page] * page + at % page).cuda()
    old_k, old_v = b.k[0][pos].to(b.q.dtype), b.v[0][pos].to(b.q.dtype)
    b.cache.write((old_k if k is None else k.to(b.q.dtype).cuda()).contiguous(),
                  (old_v if v is None else v.to(b.q.dtype).cuda()).contiguous(), slots)
    if k is not None:
        b.k[0][pos] = _held(b, b.cache.k, b.cache.k_scale, slots, page)
    if v is not None:
        b.v[0][pos] = _held(b, b.cache.v, b.cache.v_scale, slots, page)


def _exact(b, window):
    """(outputs, sizes, log sums, whether a row sees a value that is not finite in an element) in 64 bits."""
    n, t, group = b.new[0], b.total[0], b.heads // b.kv_heads
    pos, here = torch.arange(t, device="cuda"), torch.arange(n, device="cuda") + (t - n)
    seen = pos[None] <= here[:, None]
    if window:
        seen &= pos[None] > here[:, None] - window
    k, v = b.k[0].repeat_interleave(group, 1), b.v[0].repeat_interleave(group, 1)
    s = torch.einsum("ihd,jhd->hij", b.q.double(), k) / math.sqrt(b.dim)
    s = s.masked_fill(~seen[None], float("-inf"))
    p = torch.softmax(s, -1)
    bad = ~torch.isfinite(v)
    fine = torch.where(bad, 0.0, v)
    out = torch.einsum("hij,jhd->ihd", p, fine)
    size = torch.einsum("hij,jhd->ihd", p, fine.abs())
    hit = torch.einsum("ij,jhd->ihd", seen.double(), bad.double()) > 0
    return out, size, torch.logsumexp(s, -1).T, hit


def _check(b, window):
    out, lse = b.run(return_lse=True, window=window)
    want, size, want_lse, hit = _exact(b, window)
    tol = _bound(b.q.dtype, b.cache.scheme)
    top = torch.finfo(b.q.dtype).max
    over = ~hit & (want.abs() > top)
    near = ~hit & ~over & (size <= top / 2)
    assert torch.isfinite(out[near]).all(), f"{(~torch.isfinite(out[near])).sum()} of {near.sum()} not finite"
    gap = (out.double() - want).abs()[near] / (size[near] + 1e-30)
    assert (gap <= tol).all(), gap.max()
    assert (~torch.isfinite(out[hit])).all()
    assert (out[over].double() == want[over].sign() * float("inf")).all()
    assert ((lse.double() - want_lse).abs() <= 1e-4).all()


def _odd_values(b, pos, kind):
    v = b.v[0][pos].clone()
    if kind == "inf":
        v[..., 3] = float("inf")
        v[..., b.dim - 1] = float("-inf")
    elif kind == "nan":
        v[..., 5] = float("nan")
    else:
        v *= kind
    return v


@pytest.mark.parametrize("kind", ["inf", "nan", 2.0 ** 24, 2.0 ** 100])
@pytest.mark.parametrize("scheme", [None, "fp8_row", "int8_row", "mxfp4"])
@pytest.mark.parametrize("new,total,heads,kv_heads,window", SHAPES)
def test_hidden_values_leave_a_row_alone(scheme, kind, new, total, heads, kv_heads, window):
    """Keys outside the window of the first row, later tokens of the chunk: none of the rows compared sees them."""
    b = Batch([new], [total], heads, kv_heads, 128, 16, scheme, torch.bfloat16, seed=new)
    first = total - new
    hidden = [first - window - 1, first - window - 20] if window else []
    if new > 1:
        hidden.append(total - 1)
    clean = b.v[0].clone()
    _put(b, hidden, v=_odd_values(b, hidden, kind))
    b.v[0] = clean
    rows = slice(0, max(1, new - 1))
    out, lse = b.run(return_lse=True, window=window)
    want, size, want_lse, _ = _exact(b, window)
    assert torch.isfinite(out[rows]).all()
    gap = (out.double() - want).abs()[rows] / size[rows]
    assert (gap <= _bound(torch.bfloat16, scheme)).all(), gap.max()
    assert ((lse.double() - want_lse)[rows].abs() <= 1e-4).all()


@pytest.mark.parametrize("factor", [2.0 ** 12, 2.0 ** 24, 2.0 ** 60])
@pytest.mark.parametrize("scheme", ["fp8_row", "int8_row", "mxfp4"])
@pytest.mark.parametrize("new,total", [(1, 700), (4, 700), (100, 700), (1100, 1200)])
def test_a_seen_key_of_large_values_and_little_weight(scheme, factor, new, total):
    """Queries of one direction and a key far on its other side: its values count for nothing, however large."""
    b = Batch([new], [total], 1, 1, 64, 16, scheme, torch.float16 if factor < 2.0 ** 14 else torch.bfloat16, seed=new)
    u = torch.randn(64, generator=torch.Generator().manual_seed(3)).sign()
    b.q = (u * 1.5 * (1 + torch.arange(new) / (4 * new))[:, None, None]).to(b.q.dtype).cuda()
    weight = 40.0 + math.log(factor)
    _put(b, [17], k=(-u * weight / 1.5 / 8)[None, None], v=b.v[0][[17]] * factor)
    _check(b, 0)


@pytest.mark.parametrize("scheme", ["fp8_row", "int8_row", "mxfp4"])
@pytest.mark.parametrize("new,total,heads,kv_heads,window", SHAPES)
@pytest.mark.parametrize("size", [1e-2, 1e-5, 1e-9])
def test_rows_of_zeros_among_small_values(scheme, size, new, total, heads, kv_heads, window):
    """A row of zeros has a scale of its own (1): it is no measure of the others."""
    b = Batch([new], [total], heads, kv_heads, 128, 16, scheme, torch.bfloat16, seed=new)
    everything = list(range(total))
    v = b.v[0] * size
    v[::7] = 0
    v[0] = -v[0]  # zeros of either sign
    v[-3:] = 0
    _put(b, everything, v=v)
    _check(b, window)


@pytest.mark.parametrize("kind", ["inf", "nan"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16], ids=str)
@pytest.mark.parametrize("scheme", [None, "fp8_row", "int8_row", "mxfp4"])
@pytest.mark.parametrize("new,total,heads,kv_heads,window", SHAPES)
def test_seen_values_that_are_not_finite_reach_their_elements(scheme, dtype, kind, new, total, heads, kv_heads, window):
    """In units that some rows see and others do not, and in one that all see; sums and other elements stay."""
    for odd in (sorted({total - new, max(total - 40, total - new), total - 1}), [130] if not window else [total - 30]):
        b = Batch([new], [total], heads, kv_heads, 128, 16, scheme, dtype, seed=new)
        _put(b, odd, v=_odd_values(b, odd, kind))
        _check(b, window)


@pytest.mark.parametrize("scheme", [None, "fp8_row", "mxfp4"])
@pytest.mark.parametrize("new,total,heads,kv_heads", [s[:4] for s in SHAPES[1:4]])
def test_keys_that_are_not_numbers(scheme, new, total, heads, kv_heads):
    """Rows that see one are not numbers, the others are as without it."""
    b = Batch([new], [total], heads, kv_heads, 64, 16, scheme, torch.bfloat16, seed=new)
    clean = b.k[0].clone()
    at = total - new // 2
    k = b.k[0][[at]].clone()
    k[..., 7] = float("nan")
    _put(b, [at], k=k)
    b.k[0] = clean
    out, lse = b.run(return_lse=True)
    want, size, want_lse, _ = _exact(b, 0)
    rows = at - (total - new)
    assert torch.isnan(out[rows:]).all() and torch.isnan(lse[rows:]).all()
    assert ((out.double() - want).abs()[:rows] <= _bound(torch.bfloat16, scheme) * size[:rows]).all()
    assert ((lse.double() - want_lse)[:rows].abs() <= 1e-4).all()


@pytest.mark.parametrize("scheme", ["fp8_row", "int8_row", "mxfp4"])
@pytest.mark.parametrize("size", [1e-18, 1e-25, 1e-29])
@pytest.mark.parametrize("new,total,heads,kv_heads,window", SHAPES)
def test_tiny_values(scheme, size, new, total, heads, kv_heads, window):
    """What bf16 holds of them an output holds too."""
    b = Batch([new], [total], heads, kv_heads, 128, 16, scheme, torch.bfloat16, seed=new)
    _put(b, list(range(total)), v=b.v[0] * size)
    _check(b, window)


@pytest.mark.parametrize("scheme", ["fp8_row", "int8_row", "mxfp4"])
@pytest.mark.parametrize("low,high", [(2.0 ** -60, 2.0 ** 20), (2.0 ** -85, 2.0 ** 35), (2.0 ** -85, 2.0 ** 60)])
@pytest.mark.parametrize("new,total", [(1, 3000), (4, 3000), (100, 3000), (1100, 3000)])
def test_parts_of_different_sizes_weigh_the_same(scheme, low, high, new, total):
    """One stretch of the context has tiny values, the other large ones, in either order: the tiny ones' weights count in
    the sum although their values count for nothing."""
    for order in (1, -1):
        b = Batch([new], [total], 1, 1, 64, 16, scheme, torch.bfloat16, seed=new, q_scale=0.5)
        v = b.v[0]
        half = torch.arange(total, device="cuda")[:, None, None] < 1700
        v = torch.where(half if order > 0 else ~half, v * low, v * high)
        _put(b, list(range(total)), v=v)
        _check(b, 0)
