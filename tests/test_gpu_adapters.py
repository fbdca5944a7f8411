"""Low-rank adapters against the formula in 64 bits."""

from __future__ import annotations

import pytest
import torch

from tricast_b200 import get_scheme, low_rank_add, quantize, rms_norm_quantize
from tricast_b200.operand import QTensor

pytestmark = pytest.mark.gpu

HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}  # half a step: |error| / |value|


def close(out, y, x, a, b, index, gain=None):
    """Within the output's rounding, and what fp32 sums may lose: a product's sum goes through k / 16 (rank / 16) steps
    and a few dozen more where parts meet, each off by a step of the sum of magnitudes; what the lower part of a split
    intermediate leaves out is 2**-16 of it where outputs have 16 bits."""
    y, x, a, b = y.double(), x.double(), a.double(), b.double()
    ok = (index >= 0) & (index < a.shape[0])
    i = index.long().clamp(0, max(a.shape[0] - 1, 0))
    want, size = y.clone(), torch.zeros_like(y)
    for t in range(y.shape[0]):
        if ok[t]:
            h, hs = a[i[t]] @ x[t], a[i[t]].abs() @ x[t].abs()
            f = 1.0 if gain is None else gain[i[t]].double()
            want[t] += f * (b[i[t]] @ h)
            size[t] = abs(f) * (b[i[t]].abs() @ hs)
    split = 0.0 if out.dtype == torch.float32 else 2.0 ** -16
    loss = ((x.shape[1] + b.shape[2]) / 16 + 32) * 2.0 ** -23 + split
    limit = HALF[out.dtype] * (want.abs() + loss * size) + loss * size + 1e-30
    if out.dtype == torch.float16:
        limit += 2.0 ** -25  # subnormal results
    assert torch.isfinite(out).all()
    worst = ((out.double() - want).abs() / limit).max().item() if out.numel() else 0.0
    assert worst <= 1.0, worst


def inputs(tokens, k, n, rank, adapters, dtype, y_dtype, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def randn(*shape, scale=1.0):
        return torch.randn(*shape, generator=g, device="cuda") * scale

    index = torch.randint(-1, adapters + 1, (tokens,), generator=g, device="cuda").to(torch.int32)  # -1 and `adapters`: none
    return (randn(tokens, n).to(y_dtype), randn(tokens, k).to(dtype), randn(adapters, rank, k, scale=k ** -0.5).to(dtype),
            randn(adapters, n, rank, scale=0.3).to(dtype), index, 0.5 + torch.rand(adapters, generator=g, device="cuda"))


SIZES = [(1, 64, 64, 8, 1), (1, 4096, 1024, 16, 3), (2, 1, 1, 1, 2), (3, 7, 5, 3, 2), (5, 72, 40, 8, 4), (7, 1000, 264, 12, 9),
         (8, 512, 512, 64, 40), (9, 136, 1032, 24, 2), (16, 520, 1544, 40, 5), (17, 64, 72, 16, 3), (33, 333, 129, 20, 4),
         (64, 2048, 640, 32, 64), (65, 256, 200, 128, 3), (100, 96, 96, 200, 4), (257, 1024, 512, 16, 6), (600, 320, 1288, 16, 2),
         (1100, 128, 2064, 8, 5)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("size", SIZES)
def test_sizes(size, dtype):
    y, x, a, b, index, gain = inputs(*size, dtype, torch.float32)
    for out in {torch.float32, dtype}:
        close(low_rank_add(y, x, a, b, index, gain=gain, dtype=out), y, x, a, b, index, gain)
    y = y.to(dtype)
    got = low_rank_add(y, x, a, b, index)
    assert got.dtype == dtype
    close(got, y, x, a, b, index)


@pytest.mark.parametrize("order", ["runs", "alternating", "one", "none", "distinct", "blocks"])
@pytest.mark.parametrize("tokens", [1, 8, 40, 130, 700])
def test_orders_of_tokens(order, tokens):
    y, x, a, b, _, gain = inputs(tokens, 256, 328, 16, 64, torch.bfloat16, torch.float32, seed=tokens)
    t = torch.arange(tokens, device="cuda")
    index = {"runs": t // 37 % 64, "alternating": t % 2 * 63, "one": t * 0 + 5, "none": t * 0 - 1, "distinct": t % 64,
             "blocks": t // 8 % 3 - 1}[order].to(torch.int32)
    close(low_rank_add(y, x, a, b, index, gain=gain), y, x, a, b, index, gain)
    if order == "none":
        assert torch.equal(low_rank_add(y, x, a, b, index), y)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rank", [8, 16, 24, 40, 64, 96, 128])
def test_ranks_of_many_tokens(rank, dtype):
    """Stretches without an adapter, with one, and with several, beside one another."""
    y, x, a, b, index, gain = inputs(700, 264, 200, rank, 5, dtype, torch.float32, seed=rank)
    t = torch.arange(700, device="cuda")
    index = torch.where(t < 150, -1, torch.where(t < 350, 2, torch.where(t < 500, t % 7 - 1, index))).to(torch.int32)
    for out in (torch.float32, dtype):
        close(low_rank_add(y, x, a, b, index, gain=gain, dtype=out), y, x, a, b, index, gain)


@pytest.mark.parametrize("scheme", ["fp8_row", "int8_row", "fp8_e5m2"])
@pytest.mark.parametrize("tokens, k, n, rank", [(1, 512, 264, 16), (20, 1024, 512, 8), (300, 328, 640, 32), (13, 45, 19, 5)])
def test_operands_of_the_projection(scheme, tokens, k, n, rank):
    """The norm's 8-bit QTensor, and quantize's with values in a container."""
    y, x, a, b, index, gain = inputs(tokens, k, n, rank, 3, torch.bfloat16, torch.float32, seed=k)
    spec = get_scheme("fp8_row").with_(format="fp8_e5m2") if scheme == "fp8_e5m2" else get_scheme(scheme)
    normed, _ = rms_norm_quantize(x, None, spec)
    stored = quantize(x, spec)
    for q in (normed, stored):
        value = q.values.double() * q.scale.double()
        for out in (torch.float32, torch.bfloat16):
            close(low_rank_add(y, q, a, b, index, gain=gain, dtype=out), y, value, a, b, index, gain)


def test_strides_and_offsets():
    """Rows of wider tensors, at every alignment of their beginning."""
    for shift in (0, 1, 2, 4, 8):
        y, x, a, b, index, gain = inputs(50, 128 + 40, 256 + 72, 16, 3, torch.bfloat16, torch.float32, seed=shift)
        ys, xs = y[:, shift:shift + 256], x[:, shift:shift + 128]
        a, b = a[:, :, :128].contiguous(), b[:, :256].contiguous()
        close(low_rank_add(ys, xs, a, b, index, dtype=torch.bfloat16), ys, xs, a, b, index)
    y, x, a, b, index, gain = inputs(50, 128, 256, 16, 3, torch.bfloat16, torch.float32)
    close(low_rank_add(y.t().contiguous().t(), x.t().contiguous().t(), a, b, index), y, x, a, b, index)
    every = torch.stack((index, index), 1)[:, 0]
    close(low_rank_add(y[:1].expand(50, 256), x[:1].expand(50, 128), a, b, every), y[:1].expand(50, 256), x[:1].expand(50, 128),
          a, b, index)


def test_empty():
    y, x, a, b, index, _ = inputs(4, 64, 64, 8, 2, torch.bfloat16, torch.float32)
    assert low_rank_add(y[:0], x[:0], a, b, index[:0]).shape == (0, 64)
    assert torch.equal(low_rank_add(y, x, a[:0], b[:0], index), y)
    assert torch.equal(low_rank_add(y, x[:, :0], a[:, :, :0].contiguous(), b, index), y)
    assert low_rank_add(y[:, :0], x, a, b[:, :0].contiguous(), index).shape == (4, 0)


def test_values_of_other_tokens_stay_out():
    """What is not finite in one token, adapter or gain reaches no other token."""
    for tokens in (9, 64, 500):
        y, x, a, b, _, gain = inputs(tokens, 128, 192, 16, 4, torch.bfloat16, torch.float32)
        index = (torch.arange(tokens, device="cuda") % 4 - 1).to(torch.int32)  # -1, 0, 1, 2: adapter 3 is used by nobody
        a[3], b[3], gain[3] = float("nan"), float("inf"), float("nan")
        a[1, 0, 0] = float("inf")
        b[2, 5, 2] = float("nan")
        x[2] = float("nan")  # adapter 1's
        x[4, 7] = float("inf")  # no adapter's
        got = low_rank_add(y, x, a, b, index, gain=gain)
        fine = (index == 0) | (index == -1)
        clean = [t.clone() for t in (x, a, b, gain)]
        for t in clean:
            t[~torch.isfinite(t)] = 0
        want = low_rank_add(y, *clean[:3], index, gain=clean[3])
        assert torch.equal(got[fine], want[fine])
        assert torch.isnan(got[2]).all()
        col = torch.arange(192, device="cuda") != 5
        assert torch.equal(got[3][col], want[3][col]) and torch.isnan(got[3, 5])


def test_results_do_not_depend_on_the_neighbours():
    """A token's output is the same in any batch that runs the same kernel, and from call to call."""
    y, x, a, b, index, gain = inputs(400, 256, 512, 16, 6, torch.bfloat16, torch.float32)
    got = low_rank_add(y, x, a, b, index, gain=gain)
    for _ in range(3):
        assert torch.equal(got, low_rank_add(y, x, a, b, index, gain=gain))


def test_streams_and_graphs():
    y, x, a, b, index, gain = inputs(64, 256, 512, 16, 6, torch.bfloat16, torch.float32)
    want = low_rank_add(y, x, a, b, index, gain=gain)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        got = low_rank_add(y, x, a, b, index, gain=gain)
    stream.synchronize()
    assert torch.equal(got, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = low_rank_add(y, x, a, b, index, gain=gain)
    x.copy_(x.flip(0))
    index.copy_(index.flip(0))
    y.copy_(y.flip(0))
    graph.replay()
    assert torch.equal(got, low_rank_add(y, x, a, b, index, gain=gain)) and not torch.equal(got, want)


@pytest.mark.parametrize("tokens", [200, 600])
def test_captured_calls_that_share_a_stream_replay(tokens):
    """Both forms, one kernel and two, twice in one graph: each call has a workspace of its own."""
    y, x, a, b, index, gain = inputs(tokens, 256, 512, 16, 6, torch.bfloat16, torch.float32, seed=tokens)
    want = low_rank_add(y, x, a, b, index, gain=gain, dtype=torch.bfloat16)
    other = low_rank_add(y, x.flip(0), a, b, index, dtype=torch.bfloat16)
    flipped = x.flip(0)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        one = low_rank_add(y, x, a, b, index, gain=gain, dtype=torch.bfloat16)
        two = low_rank_add(y, flipped, a, b, index, dtype=torch.bfloat16)
    for _ in range(3):
        one.zero_()
        two.zero_()
        graph.replay()
        assert torch.equal(one, want) and torch.equal(two, other)


def test_calls_on_two_streams_at_once():
    sets = [inputs(700, 512, 768, 16, 6, torch.bfloat16, torch.float32, seed=s) for s in range(2)]
    want = [low_rank_add(*v[:5], gain=v[5]) for v in sets]
    streams = [torch.cuda.Stream() for _ in sets]
    torch.cuda.synchronize()
    for _ in range(10):
        got = []
        for v, stream in zip(sets, streams):
            with torch.cuda.stream(stream):
                got.append(low_rank_add(*v[:5], gain=v[5]))
        torch.cuda.synchronize()
        assert all(torch.equal(g, w) for g, w in zip(got, want))


def test_types_that_do_not_meet_in_a_product():
    """Operands of two 16-bit types, or a wide weight: element by element, the same definition."""
    y, x, a, b, index, gain = inputs(40, 96, 130, 8, 3, torch.bfloat16, torch.float32)
    close(low_rank_add(y, x.half(), a, b, index, gain=gain), y, x.half(), a, b, index, gain)
    close(low_rank_add(y, x, a.float(), b.float(), index, gain=gain), y, x, a, b, index, gain)
    close(low_rank_add(y.half(), x, a, b, index, gain=gain), y.half(), x, a, b, index, gain)
    close(low_rank_add(y, x, a, b, index, gain=gain, dtype=torch.float16), y, x, a, b, index, gain)


def test_large_and_small_products_in_fp16():
    """h beyond fp16's range, and far below it, in one batch: a token's parts have a power of two of their own."""
    for tokens in (9, 400):
        y, x, a, b, index, gain = inputs(tokens, 128, 192, 16, 3, torch.float16, torch.float32)
        x[0::3] *= 2000.0
        a[0] *= 100.0
        x[1::3] *= 2.0 ** -12
        b = b * 2.0 ** -6
        close(low_rank_add(y, x, a, b, index, gain=gain), y, x, a, b, index, gain)


def test_refusals():
    y, x, a, b, index, gain = inputs(4, 64, 96, 8, 2, torch.bfloat16, torch.float32)
    for kw in (dict(x=x[:3]), dict(x=x[:, :32]), dict(x=x[0]), dict(a=a[0]), dict(b=b[:1]), dict(b=b[:, :95]), dict(b=b.float()),
               dict(a=a.transpose(1, 2).contiguous().transpose(1, 2)), dict(index=index.long()), dict(index=index[:3]),
               dict(index=index.cpu()), dict(gain=gain[:1]), dict(gain=gain.double()), dict(x=x.double()),
               dict(y=y.double()), dict(dtype=torch.float64), dict(x=x.to(torch.int8))):
        args = dict(y=y, x=x, a=a, b=b, index=index) | kw
        with pytest.raises(ValueError):
            low_rank_add(**args)
    with pytest.raises(ValueError, match="rank"):
        low_rank_add(y, x, a.repeat(1, 200, 1), b.repeat(1, 1, 200), index)
    for scheme in ("mxfp8_e4m3", "fp8_tensor", "kivi4"):
        with pytest.raises(NotImplementedError):
            low_rank_add(y, quantize(x, scheme), a, b, index)
    with pytest.raises(NotImplementedError):
        low_rank_add(y, QTensor(x, None, None, None, get_scheme("fp8_row"), x.shape), a, b, index)
