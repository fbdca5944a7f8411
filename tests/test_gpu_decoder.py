"""The operators of a serving step together: layers with adapters, the feed-forward layer, and a decoder from request lengths to
tokens."""

from __future__ import annotations

import pytest
import torch

from tricast_b200 import (PagedKVCache, gated_quantize, gemm, get_preset, low_rank_add, paged_attention, plan_pages, quantize,
                          rms_norm_quantize, sample_tokens)
from tricast_b200.serving import Adapters, AttentionLayer, Decoder, FeedForwardLayer, generate, random_decoder, run


def test_weight_shapes_are_checked():
    ones = torch.ones
    with pytest.raises(ValueError, match="w_gate_up"):
        FeedForwardLayer(ones(96, 32), ones(32, 64), ones(32))
    with pytest.raises(ValueError, match="prompts"):
        decoder = Decoder.__new__(Decoder)
        decoder.gain = ones(4)
        generate(decoder, [[1], []], 3)


def randn_of(seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return lambda *shape, scale=0.2, dtype=torch.bfloat16: (torch.randn(*shape, generator=g, device="cuda") * scale).to(dtype)


SPEC = get_preset("nvidia_hopper_fp8").with_(out_format="fp32")


@pytest.mark.gpu
@pytest.mark.parametrize("scheme", [None, "fp8_row", "mxfp4"])
def test_run_is_what_it_was_with_tables_of_its_own(scheme):
    """The walk over prompts and steps with tables and slots made by hand: pages lie elsewhere, results are the same bits."""
    prompts, steps, hidden, heads, kv_heads, page = (200, 37), 4, 512, 8, 2, 16
    g = torch.Generator(device="cuda").manual_seed(0)

    def randn(*shape, scale=1.0):
        return (torch.randn(*shape, generator=g, device="cuda") * scale).bfloat16()

    dim, n = hidden // heads, len(prompts)
    layer = AttentionLayer(randn((heads + 2 * kv_heads) * dim, hidden, scale=hidden ** -0.5), randn(hidden, hidden, scale=hidden ** -0.5),
                           torch.ones(hidden, dtype=torch.bfloat16, device="cuda"), heads, kv_heads)
    pages = -(-(max(prompts) + steps) // page)
    cache = PagedKVCache(n * pages, page, kv_heads, dim, scheme)
    table = torch.randperm(n * pages, generator=g, device="cuda").to(torch.int32).view(n, pages)

    def slots(seq, first, count):
        at = torch.arange(first, first + count, device="cuda")
        return table[seq, at // page].long() * page + at % page

    lens = torch.tensor(prompts, dtype=torch.int32, device="cuda")
    cu = torch.nn.functional.pad(lens.cumsum(0), (1, 0)).to(torch.int32)
    where = torch.cat([slots(i, 0, p) for i, p in enumerate(prompts)])
    x, residual = randn(sum(prompts), hidden), randn(sum(prompts), hidden)
    want = [layer(x, residual, cache, where, table, lens, cu, max_q_len=max(prompts))[0]]
    for t in range(steps):
        where = torch.cat([slots(i, p + t, 1) for i, p in enumerate(prompts)])
        x, residual = randn(n, hidden), randn(n, hidden)
        want.append(layer(x, residual, cache, where, table, lens + t + 1)[0])
    for a, b in zip(run(scheme), want):
        assert torch.equal(a, b)


@pytest.mark.gpu
@pytest.mark.parametrize("scheme", ["fp8_row", "int8_row", "fp8_group128"])
def test_a_feed_forward_call_is_its_operators_in_turn(scheme):
    randn = randn_of(1)
    up, down, gain = randn(2 * 320, 128), randn(128, 320), randn(128)
    x, r = randn(21, 128), randn(21, 128)
    out, h = FeedForwardLayer(up, down, gain, scheme=scheme, activation="gelu_tanh")(x, r)
    normed, want_h = rms_norm_quantize(x, gain, scheme, residual=r)
    y = gemm(normed, quantize(up, scheme), SPEC)
    gated = gated_quantize(y[:, :320], y[:, 320:], scheme, activation="gelu_tanh")
    want = gemm(gated, quantize(down, scheme), SPEC).bfloat16()
    assert torch.equal(out, want) and torch.equal(h, want_h)
    alone, same = FeedForwardLayer(up, down, gain, scheme=scheme)(x, None)
    assert same is x and torch.isfinite(alone).all()


@pytest.mark.gpu
def test_adapters_stand_beside_both_projections():
    randn = randn_of(2)
    wq, wo, gain = randn(8 * 32, 128), randn(128, 4 * 32), randn(128)
    up, down = randn(2 * 192, 128), randn(128, 192)
    beside = {"qkv": Adapters(randn(3, 8, 128), randn(3, 256, 8), torch.tensor([1.0, 0.5, 2.0], device="cuda")),
              "out": Adapters(randn(3, 4, 128), randn(3, 128, 4)), "up": Adapters(randn(3, 16, 128), randn(3, 384, 16)),
              "down": Adapters(randn(3, 16, 192), randn(3, 128, 16))}
    attention = AttentionLayer(wq, wo, gain, 4, 2, qkv_adapters=beside["qkv"], out_adapters=beside["out"])
    forward = FeedForwardLayer(up, down, gain, gate_up_adapters=beside["up"], down_adapters=beside["down"])
    x, r = randn(9, 128), randn(9, 128)
    table = torch.tensor([[1, 0]], dtype=torch.int32, device="cuda")
    slots = torch.cat([torch.arange(8, 16), torch.arange(1)]).cuda()
    lens, cu = torch.tensor([9], dtype=torch.int32, device="cuda"), torch.tensor([0, 9], dtype=torch.int32, device="cuda")
    index = torch.tensor([0, 0, -1, 2, 1, 1, -1, 0, 2], dtype=torch.int32, device="cuda")

    def add(y, operand, which):
        a, b, factor = beside[which]
        return low_rank_add(y, operand, a, b, index, gain=factor, dtype=torch.bfloat16)

    out, h = attention(x, r, PagedKVCache(2, 8, 2, 32), slots, table, lens, cu, max_q_len=9, index=index)
    normed, _ = rms_norm_quantize(x, gain, "fp8_row", residual=r)
    qkv = add(gemm(normed, quantize(wq, "fp8_row"), SPEC), normed, "qkv").view(9, 8, 32)
    cache = PagedKVCache(2, 8, 2, 32)
    cache.write(qkv[:, 4:6], qkv[:, 6:], slots)
    a = paged_attention(qkv[:, :4], cache, table, lens, cu, max_q_len=9).view(9, 128)
    assert torch.equal(out, add(gemm(quantize(a, "fp8_row"), quantize(wo, "fp8_row"), SPEC), a, "out"))
    got, _ = forward(x, r, index=index)
    y = add(gemm(normed, quantize(up, "fp8_row"), SPEC), normed, "up")
    gated = gated_quantize(y[:, :192], y[:, 192:], "fp8_row")
    assert torch.equal(got, add(gemm(gated, quantize(down, "fp8_row"), SPEC), gated, "down"))
    # No adapter for anyone is the layer without adapters.
    nobody = torch.full_like(index, -1)
    for layer, plain in ((attention, AttentionLayer(wq, wo, gain, 4, 2)),):
        args = (slots, table, lens, cu)
        assert torch.equal(layer(x, r, PagedKVCache(2, 8, 2, 32), *args, index=nobody)[0], plain(x, r, PagedKVCache(2, 8, 2, 32), *args)[0])


@pytest.mark.gpu
def test_a_step_at_a_time_is_the_whole_prompt_at_once():
    """In fp32 every row of every operator is computed by itself: what the cache and the plan hold after steps gives the bits of a
    prompt that has those tokens from the start."""
    decoder = random_decoder(vocab=300, hidden=64, heads=2, kv_heads=1, inner=96, dtype=torch.float32, adapters=2, seed=3)
    prompts, steps = [[5, 9, 2], [7] * 18, [1]], 6
    uniform = torch.rand(steps, 3, generator=torch.Generator().manual_seed(2)).cuda()
    adapter = torch.tensor([1, -1, 0], dtype=torch.int32, device="cuda")
    settings = dict(adapter=adapter, temperature=0.8, top_k=40, top_p=0.9)
    said = generate(decoder, prompts, steps, None, uniform=uniform, page_size=8, **settings)
    assert said.shape == (3, steps) and ((said >= 0) & (said < 300)).all()
    assert torch.equal(said, generate(decoder, prompts, steps, None, uniform=uniform, page_size=16, **settings))
    for t in range(1, steps):
        longer = [p + said[i, :t].tolist() for i, p in enumerate(prompts)]
        assert torch.equal(generate(decoder, longer, 1, None, uniform=uniform[t:], **settings)[:, 0], said[:, t])


@pytest.mark.gpu
def test_a_captured_decode_step_replays():
    """Plan, layers with adapters and sampling in one graph: replays go on where the eager steps would."""
    decoder = random_decoder(vocab=500, hidden=64, heads=2, kv_heads=1, inner=128, adapters=3, seed=4)
    prompts, steps = [[3, 1, 4, 1, 5], [9] * 11], 9
    uniform = torch.rand(steps, 2, generator=torch.Generator().manual_seed(5)).cuda()
    adapter = torch.tensor([2, 0], dtype=torch.int32, device="cuda")
    want = generate(decoder, prompts, steps, "fp8_row", uniform=uniform, page_size=8, adapter=adapter, top_p=0.9)
    as32 = dict(dtype=torch.int32, device="cuda")
    caches = [PagedKVCache(8, 8, a.kv_heads, a.head_dim, "fp8_row", dtype=a.dtype) for a, _ in decoder.layers]
    table, free, taken, have = torch.full((2, 4), -1, **as32), torch.arange(8, **as32), torch.zeros(1, **as32), torch.zeros(2, **as32)
    plan = plan_pages(have, torch.tensor([5, 11], **as32), table, free, taken, page_size=8, tokens=16)
    first = torch.tensor([t for p in prompts for t in p], device="cuda")
    logits = decoder(first, caches, plan, table, max_q_len=11, index=adapter[plan.sequence.long()])
    tokens = sample_tokens(logits, uniform[0], top_p=0.9)
    got = [tokens.clone()]
    have.copy_(plan.seq_lens)
    taken.copy_(plan.taken)
    one, u = torch.ones(2, **as32), uniform[1].clone()

    def step():
        p = plan_pages(have, one, table, free, taken, page_size=8, tokens=2)
        t = sample_tokens(decoder(tokens, caches, p, table, max_q_len=1, index=adapter[p.sequence.long()]), u, top_p=0.9)
        tokens.copy_(t)
        have.copy_(p.seq_lens)
        taken.copy_(p.taken)

    step()  # warms up, and is the second step
    got.append(tokens.clone())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for t in range(2, steps):
        u.copy_(uniform[t])
        graph.replay()
        got.append(tokens.clone())
    assert torch.equal(torch.stack(got, 1), want)
