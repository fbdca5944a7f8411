"""The attention layer that runs the serving operators together."""

from __future__ import annotations

import pytest
import torch

from tricast_b200 import PagedKVCache, gemm, get_preset, paged_attention, quantize, rms_norm_quantize
from tricast_b200.serving import AttentionLayer, run


def test_weight_shapes_are_checked():
    ones = torch.ones
    with pytest.raises(ValueError, match="multiple"):
        AttentionLayer(ones(96, 32), ones(32, 48), ones(32), 3, 2)
    with pytest.raises(ValueError, match="w_qkv"):
        AttentionLayer(ones(80, 32), ones(32, 48), ones(32), 4, 2)


@pytest.mark.gpu
def test_a_call_is_its_operators_in_turn():
    g = torch.Generator(device="cuda").manual_seed(3)

    def randn(*shape):
        return (torch.randn(*shape, generator=g, device="cuda") * 0.2).bfloat16()

    wq, wo, gain = randn((4 + 2 * 2) * 32, 128), randn(128, 4 * 32), randn(128)
    layer = AttentionLayer(wq, wo, gain, 4, 2)
    x, r = randn(9, 128), randn(9, 128)
    table = torch.tensor([[1, 0]], dtype=torch.int32, device="cuda")
    slots = torch.cat([torch.arange(8, 16), torch.arange(1)]).cuda()
    lens, cu = torch.tensor([9], dtype=torch.int32, device="cuda"), torch.tensor([0, 9], dtype=torch.int32, device="cuda")
    caches = [PagedKVCache(2, 8, 2, 32, "int8_row") for _ in range(2)]
    out, h = layer(x, r, caches[0], slots, table, lens, cu, max_q_len=9)
    spec = get_preset("nvidia_hopper_fp8").with_(out_format="fp32")
    normed, want_h = rms_norm_quantize(x, gain, "fp8_row", residual=r)
    qkv = gemm(normed, quantize(wq, "fp8_row"), spec).bfloat16().view(9, 8, 32)
    caches[1].write(qkv[:, 4:6].contiguous(), qkv[:, 6:].contiguous(), slots)
    a = paged_attention(qkv[:, :4].contiguous(), caches[1], table, lens, cu, max_q_len=9)
    want = gemm(quantize(a.view(9, 128), "fp8_row"), quantize(wo, "fp8_row"), spec).bfloat16()
    assert torch.equal(out, want) and torch.equal(h, want_h)
    alone, same = layer(x, None, caches[0], slots, table, lens, cu, max_q_len=9)
    assert same is x and torch.isfinite(alone).all()


@pytest.mark.gpu
@pytest.mark.parametrize("scheme,db", [("fp8_row", 12.0), ("int8_row", 12.0), ("mxfp4", 3.0)])
def test_prompts_and_steps_follow_the_unquantized_cache(scheme, db):
    """E4M3 rounds within 2**-4 of an element, so V's part alone leaves 24 dB at the worst, and K's, whose scores are of
    order 1, and the 8-bit GEMM operand's as much again: 12 dB. INT8 rows are finer. E2M1 rounds within 2**-2: 3 dB."""
    for want, got in zip(run(None), run(scheme)):
        assert torch.isfinite(got).all()
        noise = (want.double() - got.double()).square().sum()
        assert 10 * torch.log10(want.double().square().sum() / noise).item() >= db
