"""The quantized paged cache: what is written equals, bit for bit, what the quantize kernels give for the
same rows, and what is read back equals their dequantization."""

from __future__ import annotations

import pytest
import torch

from tricast_b200 import PagedKVCache, quantize_into
from tricast_b200.spec import SCHEMES

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def _rows(tokens, heads, dim, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(tokens, heads, dim, generator=g)
    x[..., torch.randperm(dim, generator=g)[:2]] *= 8
    if tokens > 6:
        x[1] = 0
        x[2] *= 2.0 ** -14
        x[3, :, dim // 2] = float("nan")
        x[4, :, 0] = float("inf")
        x[5] *= 1000
    return x.to(dtype).cuda()


def _same(a, b):
    return torch.equal(torch.nan_to_num(a.float(), nan=12345.0, posinf=1e30, neginf=-1e30),
                       torch.nan_to_num(b.float(), nan=12345.0, posinf=1e30, neginf=-1e30))


def _expected(x, scheme):
    """(code bytes, scales, dequantized values) of each row from the quantize kernels."""
    t, h, d = x.shape
    if scheme is None:
        return x.view(torch.uint8), None, x
    q, extras = quantize_into(x.reshape(-1, d), SCHEMES[scheme], want_codes=True,
                              want_scale_codes=scheme == "mxfp4")
    codes = extras.codes.reshape(t, h, -1)
    scales = extras.scale_codes.reshape(t, h, -1) if scheme == "mxfp4" else q.scale.reshape(t, h)
    values = q.dequantize()
    if scheme == "int8_row":  # integer codes have no NaN: a NaN keeps code 0, and the row's scale
        s = q.scale.reshape(-1, 1)
        values = torch.where(q.values.isnan(), 0.0 * s, values)
    return codes, scales, values.reshape(t, h, d).to(x.dtype)


@pytest.mark.parametrize("scheme", [None, "fp8_row", "int8_row", "mxfp4"])
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("tokens,heads,dim,page", [(1, 1, 32, 8), (37, 3, 64, 16), (130, 8, 128, 64), (20, 2, 96, 32),
                                                   (9, 5, 256, 128), (300, 1, 160, 256)])
def test_write_and_read(scheme, dtype, tokens, heads, dim, page):
    pages = -(-tokens // page) + 2
    cache = PagedKVCache(pages, page, heads, dim, scheme, dtype=dtype)
    g = torch.Generator().manual_seed(tokens)
    slots = torch.randperm(pages * page, generator=g)[:tokens].cuda()
    k, v = _rows(tokens, heads, dim, dtype, 1), _rows(tokens, heads, dim, dtype, 2)
    cache.write(k, v, slots)
    p, o = slots // page, slots % page
    got = cache.read(slots)
    for x, pool, scales, back in ((k, cache.k, cache.k_scale, got[0]), (v, cache.v, cache.v_scale, got[1])):
        codes, s, values = _expected(x, scheme)
        here = pool.view(torch.uint8)[p, :, o]
        assert torch.equal(here, codes.reshape(here.shape))
        if s is not None:
            kept = scales.view(torch.uint8)[p, :, o] if scheme == "mxfp4" else scales[p, :, o]
            assert _same(kept, s) if scheme != "mxfp4" else torch.equal(kept, s)
        assert back.dtype == dtype and _same(back, values)
    # Nothing else was touched.
    rest = torch.ones(pages * page, dtype=torch.bool, device="cuda")
    rest[slots] = False
    free = rest.nonzero().squeeze(1)
    assert not cache.k.view(torch.uint8)[free // page, :, free % page].any()
    assert not cache.v.view(torch.uint8)[free // page, :, free % page].any()


@pytest.mark.parametrize("scheme", [None, "fp8_row", "int8_row", "mxfp4"])
def test_strided_inputs_and_skipped_slots(scheme):
    tokens, heads, dim, page = 50, 4, 64, 16
    qkv = _rows(tokens, 3 * heads, dim, torch.bfloat16, 5)
    k, v = qkv[:, heads:2 * heads], qkv[:, 2 * heads:]
    a, b = (PagedKVCache(6, page, heads, dim, scheme) for _ in range(2))
    slots = torch.randperm(96, generator=torch.Generator().manual_seed(1))[:tokens].cuda()
    some = slots.clone()
    some[::7] = -1
    some[3] = 96
    some[4] = 1 << 40
    a.write(k, v, some)
    keep = (some >= 0) & (some < 96)
    b.write(k[keep].contiguous(), v[keep].contiguous(), some[keep])
    for x, y in ((a.k, b.k), (a.v, b.v)):
        assert torch.equal(x.view(torch.uint8), y.view(torch.uint8))
    rk, rv = a.read(some)
    assert (rk[~keep] == 0).all() and (rv[~keep] == 0).all()
    ok, _ = b.read(some[keep])
    assert _same(rk[keep], ok)
    odd = _rows(tokens, heads, 2 * dim + 3, torch.bfloat16, 6)  # rows that start off any vector boundary
    a.write(odd[..., 1:dim + 1], odd[..., dim + 2:2 * dim + 2], slots)
    b.write(odd[..., 1:dim + 1].contiguous(), odd[..., dim + 2:2 * dim + 2].contiguous(), slots)
    assert _same(a.read(slots)[0], b.read(slots)[0]) and _same(a.read(slots)[1], b.read(slots)[1])
    step = _rows(tokens, heads, 2 * dim, torch.bfloat16, 7)[..., ::2]
    a.write(step, step, slots)
    b.write(step.contiguous(), step.contiguous(), slots)
    assert _same(a.read(slots)[0], b.read(slots)[0])


def test_no_tokens_and_another_stream():
    cache = PagedKVCache(2, 8, 2, 32, "fp8_row")
    none = torch.empty(0, 2, 32, device="cuda", dtype=torch.bfloat16)
    cache.write(none, none, torch.empty(0, dtype=torch.int64, device="cuda"))
    assert cache.read(torch.empty(0, dtype=torch.int64, device="cuda"))[0].shape == (0, 2, 32)
    x = _rows(16, 2, 32, torch.bfloat16, 1)
    slots = torch.arange(16, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        cache.write(x, x, slots)
        got, _ = cache.read(slots)
    torch.cuda.current_stream().wait_stream(side)
    assert _same(got, _expected(x, "fp8_row")[2])


def test_offsets_beyond_32_bits():
    """The last page of a pool of more than 2**32 bytes."""
    pages, page, heads, dim = 70000, 64, 8, 128
    cache = PagedKVCache(pages, page, heads, dim, "fp8_row")
    x = _rows(64, heads, dim, torch.bfloat16, 3)
    slots = torch.arange((pages - 1) * page, pages * page, device="cuda")
    cache.write(x, x, slots)
    assert cache.k.numel() > 2 ** 32
    got = cache.read(slots)
    want = _expected(x, "fp8_row")[2]
    assert _same(got[0], want) and _same(got[1], want)
    assert not cache.k[0].view(torch.uint8).any()


def test_refusals():
    for bad in (dict(page_size=24), dict(page_size=4), dict(page_size=512), dict(head_dim=24), dict(head_dim=512),
                dict(num_pages=0), dict(kv_heads=0)):
        args = dict(num_pages=2, page_size=16, kv_heads=2, head_dim=64) | bad
        with pytest.raises(ValueError):
            PagedKVCache(**args)
    with pytest.raises(ValueError, match="multiple of 16"):
        PagedKVCache(2, 16, 2, 48, "mxfp4")
    with pytest.raises(ValueError, match="unknown cache scheme"):
        PagedKVCache(2, 16, 2, 64, "fp8_tensor")
    with pytest.raises(ValueError, match="CUDA device"):
        PagedKVCache(2, 16, 2, 64, device="cpu")
    cache = PagedKVCache(2, 16, 2, 64)
    x = torch.zeros(4, 2, 64, device="cuda", dtype=torch.bfloat16)
    slots = torch.arange(4, device="cuda")
    for k, s in ((x.half(), slots), (x[:3], slots), (x[:, :1], slots), (x.cpu(), slots), (x, slots.int()), (x, slots.cpu()),
                 (x, slots[None])):
        with pytest.raises(ValueError):
            cache.write(k, x, s)
