"""Sampling against the definition in 64 bits, row by row."""

from __future__ import annotations

import math

import numpy as np
import pytest
import torch

from tricast_b200 import sample_tokens

pytestmark = pytest.mark.gpu

EDGE = 1e-7  # weights are good to 1.4 halves of an fp32 step (8.3e-8), so are their shares: a border this near may fall on either side


def draw(z, u, heat, k, p, m):
    """(token, log-probability, distance of the nearest border) by sorting, in 64 bits; settings as fp32 numbers."""
    if np.isnan(z).any():
        return -1, math.nan, 1.0
    if z.max() == -np.inf:
        return -1, -math.inf, 1.0
    if not heat > 0:
        return int(z.argmax()), 0.0, 1.0
    heat = max(heat, 2.0 ** -100)
    with np.errstate(invalid="ignore", over="ignore"):
        w = np.exp((z - z.max()) / heat)
    w[z == z.max()] = 1.0
    w[np.isnan(w) | (z == -np.inf) | (w < 2.0 ** -126)] = 0.0
    order = np.argsort(-z, kind="stable")
    order = order[w[order] > 0]
    near, ones = 1.0, (w[order] == 1).all()  # sums of ones, and their products with fp32 numbers, are exact: no border is near
    if k > 0:
        order = order[:k]
    if p < 1:
        upto = np.cumsum(w[order])
        short = upto < p * upto[-1]
        near = min(near, np.abs(upto / upto[-1] - p).min() / max(w[order].min() / upto[-1], 1e-3))
        order = order[: short.sum() + 1]
    if m > 0:
        keep = w[order] >= min(m, 1.0)
        near = min(near, np.abs(w[order][w[order] < 1] / m - 1).min(initial=1.0))
        order = order[keep]
    ids = np.sort(order)
    upto = np.cumsum(w[ids])
    j = min(int(np.searchsorted(upto, u * upto[-1], side="right")), len(ids) - 1)
    # The last border is the total itself, whatever it is off.
    near = 1.0 if ones else min(near, np.abs(upto[:-1] / upto[-1] - u).min(initial=1.0))
    return int(ids[j]), math.log(w[ids[j]] / upto[-1]), near


def check(logits, u, temperature=1.0, top_k=None, top_p=None, min_p=None):
    tokens, logprobs = sample_tokens(logits, u, temperature=temperature, top_k=top_k, top_p=top_p, min_p=min_p, return_logprobs=True)
    assert torch.equal(tokens, sample_tokens(logits, u, temperature=temperature, top_k=top_k, top_p=top_p, min_p=min_p))
    z, rows = logits.double().cpu().numpy(), logits.shape[0]

    def of(v, neutral):
        if v is None:
            return [neutral] * rows
        return v.double().tolist() if isinstance(v, torch.Tensor) else [float(np.float32(v))] * rows

    settings = list(zip(u.double().tolist(), of(temperature, 1.0), of(top_k, 0), of(top_p, 1.0), of(min_p, 0.0)))
    loose = 0
    for r in range(rows):
        uu, heat, k, p, m = settings[r]
        token, logprob, near = draw(z[r], uu, heat, int(k), p, m)
        if near < EDGE:
            loose += 1
            continue
        assert tokens[r].item() == token, (r, settings[r], near)
        got = logprobs[r].item()
        assert got == logprob or (math.isnan(got) and math.isnan(logprob)) or abs(got - logprob) <= 3e-6 + 2.0 ** -23 * abs(logprob), (got, logprob)
    assert loose <= max(2, rows // 10)


def make(rows, vocab, dtype=torch.float32, seed=0, spread=2.5):
    g = torch.Generator(device="cuda").manual_seed(seed + rows * vocab)
    z = (torch.randn(rows, vocab, generator=g, device="cuda") * spread).to(dtype)
    return z, torch.rand(rows, generator=g, device="cuda"), g


VOCABS = [1, 2, 3, 31, 33, 257, 1000, 4099, 16383, 16384, 16391, 40001, 70000, 131072]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("vocab", VOCABS)
def test_filters(vocab, dtype):
    z, u, g = make(12, vocab, dtype)
    for kw in (dict(), dict(top_k=1), dict(top_k=7), dict(top_k=50), dict(top_p=0.9), dict(top_p=0.3), dict(min_p=0.05),
               dict(top_k=40, top_p=0.95), dict(top_k=1000, top_p=0.99, min_p=0.001), dict(temperature=0.0),
               dict(temperature=0.7, top_p=0.999), dict(temperature=1.7, top_p=0.5, min_p=0.02), dict(temperature=0.05)):
        check(z, u, **kw)


@pytest.mark.parametrize("vocab", [100, 5000, 50257])
def test_settings_of_each_row(vocab):
    z, u, g = make(64, vocab)

    def choose(*of, dtype=torch.float32):
        return torch.tensor(of, device="cuda", dtype=dtype)[torch.randint(0, len(of), (64,), generator=g, device="cuda")]

    for _ in range(3):
        check(z, u, choose(0.0, 0.5, 1.0, 2.0, -1.0), choose(0, -3, 1, 5, 60, 4000, 10 ** 6, dtype=torch.int32),
              choose(0.0, 0.1, 0.8, 0.99, 1.0, 2.0), choose(0.0, -1.0, 0.1, 0.5, 1.0, 3.0))


@pytest.mark.parametrize("vocab", [64, 3000, 20000])
@pytest.mark.parametrize("values", [1, 2, 5])
def test_ties(vocab, values):
    """Rows of a few distinct values: filters end inside a run of equals and keep the first of them."""
    g = torch.Generator(device="cuda").manual_seed(vocab + values)
    z = torch.randint(0, values, (24, vocab), generator=g, device="cuda").bfloat16() * 0.5
    u = torch.rand(24, generator=g, device="cuda")
    for kw in (dict(), dict(top_k=3), dict(top_k=vocab // 2), dict(top_k=vocab - 1), dict(top_p=0.37), dict(top_p=0.47, top_k=vocab // 3),
               dict(top_p=1e-9), dict(min_p=0.7), dict(min_p=1.0), dict(temperature=0.0), dict(top_k=vocab)):
        check(z, u, **kw)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("vocab", [50, 2000, 33000])
def test_masks(vocab, dtype):
    """Banned tokens at -inf or at the type's lowest value; rows of nothing else, of one token, of NaN, of infinities."""
    z, u, g = make(16, vocab, dtype, seed=3)
    low = torch.finfo(dtype).min
    z[0:4, 5:] = float("-inf")
    z[4:6, 5:] = low
    z[6] = float("-inf")
    z[7] = low
    z[8, vocab // 2] = float("nan")
    z[9] = float("nan")
    z[10, [3, vocab - 1]] = float("inf")
    z[11] = float("-inf")
    z[11, vocab - 1] = low
    z[12, : vocab - 1] = float("-inf")
    z[13] = -0.0
    z[13, ::2] = 0.0
    z[14, 1] = torch.finfo(dtype).max
    z[15, torch.rand(vocab, generator=g, device="cuda") < 0.5] = float("-inf")
    for kw in (dict(), dict(top_k=3), dict(top_k=20), dict(top_p=0.9), dict(top_k=6, top_p=0.8), dict(min_p=0.1), dict(temperature=0.0),
               dict(temperature=1e30), dict(temperature=float("inf"), top_k=30), dict(temperature=1e-30, top_p=0.5),
               dict(temperature=1e-44, top_k=9)):
        check(z, u, **kw)


def test_ends_of_the_random_numbers():
    z, _, _ = make(8, 3001)
    z[:, 0] = z[:, -1] = float("-inf")
    one = 1 - 2.0 ** -24
    for v in (0.0, one, 1.0, 2.0, -1.0, float("nan")):
        u = torch.full((8,), v, device="cuda")
        for kw in (dict(), dict(top_k=5), dict(top_p=0.9)):
            t = sample_tokens(z, u, **kw)
            if not v >= 1:  # the first that is kept: no number below 0, nor NaN, leaves the row
                assert ((t > 0) & (t < 3000)).all()
            if v == 0.0 or v == one:
                check(z, u, **kw)


def test_settings_that_are_not_numbers():
    z, u, _ = make(6, 900)
    nan = float("nan")
    want = sample_tokens(z, u)
    assert torch.equal(sample_tokens(z, u, top_p=nan, min_p=nan), want)
    assert torch.equal(sample_tokens(z, u, temperature=nan), z.argmax(1))


def test_wide_and_narrow_ranges():
    """Logits far apart, all within a few steps of fp32, subnormal, and with one far above the rest."""
    g = torch.Generator(device="cuda").manual_seed(8)
    base = torch.randn(5, 30000, generator=g, device="cuda")
    u = torch.rand(5, generator=g, device="cuda")
    for z in (base * 1e4, base * 1e37, base * 1e-41, 1 + base * 1e-7, base + 1000.0, torch.cat((base, base[:, :1] * 0 + 60), 1)):
        for kw in (dict(), dict(top_k=100), dict(top_p=0.7), dict(top_k=20000, top_p=0.9), dict(min_p=0.5), dict(temperature=0.0)):
            check(z, u, **kw)


def test_flat_rows_of_many_kept_tokens():
    g = torch.Generator(device="cuda").manual_seed(9)
    z = torch.randn(6, 131072, generator=g, device="cuda") * 0.3
    u = torch.rand(6, generator=g, device="cuda")
    for kw in (dict(top_p=0.9), dict(top_k=60000), dict(top_k=60000, top_p=0.8), dict(min_p=0.2), dict(temperature=3.0, top_p=0.99)):
        check(z, u, **kw)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_large_vocabularies(dtype):
    """Beyond what a cluster's shared memory holds: weights are computed anew by every pass."""
    z, u, _ = make(2, 600001, dtype)
    z[1, 3:7] = float("-inf")
    for kw in (dict(), dict(top_k=50, top_p=0.9), dict(top_p=0.95), dict(temperature=0.0), dict(top_k=30000, top_p=0.8), dict(min_p=0.01),
               dict(temperature=float("inf"), top_k=70001)):
        check(z, u, **kw)
    z[0, 5] = z[0, 500000] = float("inf")
    z[1, 400000] = float("nan")
    check(z, u, top_p=0.9)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("min_p", [None, 1e-3])
def test_unfiltered_rows_of_large_vocabularies(dtype, min_p):
    """Weights within 1.2e-10 move a share by 2.4e-10 at most, sums of n of them in 64 bits by n 2**-53: borders nearer than 4e-10 may
    fall on either side, as may the bound. With 164724 tokens some row in ten thousand has such a border."""
    rows, vocab = 256, 164724
    z, u, g = make(rows, vocab, dtype)
    w = torch.exp(z.double() - z.double().amax(1, keepdim=True))
    if min_p is not None:
        bound = float(np.float32(min_p))
        assert not ((w / bound - 1).abs() < 1e-9).any()
        w[w < bound] = 0.0
    upto = w.cumsum(1)
    share = upto / upto[:, -1:]
    want = torch.searchsorted(share, u.double()[:, None], right=True)[:, 0].clamp(max=vocab - 1)
    near = (share[:, :-1] - u.double()[:, None]).abs().amin(1) < 4e-10
    assert near.sum() <= 1
    tokens, logprobs = sample_tokens(z, u, min_p=min_p, return_logprobs=True)
    assert torch.equal(tokens[~near], want[~near].to(tokens.dtype))
    exact = (w.gather(1, tokens[:, None].long()) / upto[:, -1:]).log()[:, 0]
    assert ((logprobs.double() - exact).abs() <= 2.0 ** -24 * exact.abs() + 1e-9).all()


@pytest.mark.parametrize("vocab", [513, 5000, 60000])
def test_sets_as_long_as_one_block_finishes(vocab):
    """Around 512 tokens, below and above which other code ends the work; runs of equals that pass it."""
    for dtype in (torch.float32, torch.bfloat16):
        z, u, _ = make(6, vocab, dtype, seed=11)
        z[4] = (z[4] > 0).to(dtype)  # two values
        z[5, 20:] = float("-inf")  # fewer tokens than top_k
        for k in (2, 31, 33, 255, 500, 511, 512, 513, 600):
            check(z, u, top_k=k)
            check(z, u, top_k=k, top_p=0.7, min_p=0.01, temperature=1.3)


def test_many_rows_and_strides():
    z, u, _ = make(700, 515)
    check(z, u, top_k=30, top_p=0.9)
    for shift in (0, 1, 3, 8):
        for dtype in (torch.float32, torch.bfloat16):
            w, u, _ = make(9, 20100, dtype, seed=shift)
            check(w[:, shift:20000 + shift], u, top_k=30, top_p=0.9)
            check(w[:, shift:20000 + shift], u)
    w, u, _ = make(9, 300)
    check(w.t().contiguous().t(), u, top_p=0.5)
    check(w[:1].expand(9, 300), u, top_p=0.5)


def test_tokens_follow_their_probabilities():
    """One row, stratified random numbers: counts are the probabilities to one token."""
    z, _, _ = make(1, 40)
    n = 4000
    u = (torch.arange(n, device="cuda") + 0.5) / n
    t = sample_tokens(z.expand(n, 40), u, top_k=20)
    w = z.double().softmax(1)[0]
    w[w.argsort(descending=True)[20:]] = 0
    want = w / w.sum() * n
    got = torch.bincount(t, minlength=40).double()
    assert (got - want).abs().max() <= 1.001


def test_streams_and_graphs():
    z, u, _ = make(20, 20000)
    want = sample_tokens(z, u, top_k=50, top_p=0.9)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        got = sample_tokens(z, u, top_k=50, top_p=0.9)
    stream.synchronize()
    assert torch.equal(got, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = sample_tokens(z, u, top_k=50, top_p=0.9)
    z.copy_(z.flip(0))
    u.copy_(u.flip(0))
    graph.replay()
    assert torch.equal(got, want.flip(0))


def test_calls_on_two_streams_at_once():
    sets = [make(40, 30000, seed=s)[:2] for s in range(2)]
    want = [sample_tokens(z, u, top_p=0.9) for z, u in sets]
    streams = [torch.cuda.Stream() for _ in sets]
    torch.cuda.synchronize()
    for _ in range(10):
        got = []
        for (z, u), stream in zip(sets, streams):
            with torch.cuda.stream(stream):
                got.append(sample_tokens(z, u, top_p=0.9))
        torch.cuda.synchronize()
        assert all(torch.equal(g, w) for g, w in zip(got, want))


def test_refusals():
    z, u, _ = make(4, 100)
    for kw in (dict(uniform=u[:3]), dict(uniform=u.double()), dict(uniform=0.5), dict(uniform=u.cpu()), dict(logits=z[0]),
               dict(logits=z[:, :0]), dict(logits=z.double()), dict(temperature=u[:2]), dict(top_k=u), dict(top_p=u.cpu()),
               dict(min_p=u.double())):
        with pytest.raises(ValueError):
            sample_tokens(**(dict(logits=z, uniform=u) | kw))
    assert sample_tokens(z[:0], u[:0]).shape == (0,)
