"""What a request gets from layers and decoders does not depend on what else is asked for."""

from __future__ import annotations

import pytest
import torch

from tricast_b200 import PagedKVCache
from tricast_b200.serving import Adapters, AttentionLayer, FeedForwardLayer


def randn_of(seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return lambda *shape, scale=0.2, dtype=torch.bfloat16: (torch.randn(*shape, generator=g, device="cuda") * scale).to(dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("activation", ["silu", "gelu_tanh"])
def test_requests_without_an_adapter_among_others(dtype, activation):
    """Layers with adapters, called without an index, with one that names nobody's adapter, and with one that names some."""
    randn = randn_of(7)
    randn = lambda *shape, f=randn: f(*shape, dtype=dtype)  # noqa: E731
    wq, wo, gain, up, down = randn(8 * 32, 128), randn(128, 4 * 32), randn(128), randn(2 * 320, 128), randn(128, 320)
    attention = AttentionLayer(wq, wo, gain, 4, 2, qkv_adapters=Adapters(randn(3, 8, 128), randn(3, 256, 8)),
                               out_adapters=Adapters(randn(3, 8, 128), randn(3, 128, 8)))
    forward = FeedForwardLayer(up, down, gain, activation=activation, gate_up_adapters=Adapters(randn(3, 8, 128), randn(3, 640, 8)),
                               down_adapters=Adapters(randn(3, 8, 320), randn(3, 128, 8)))
    x, r = randn(40, 128), randn(40, 128)
    table = torch.arange(40, dtype=torch.int32, device="cuda")[:, None]  # 40 requests of a token each
    slots, lens = torch.arange(40, device="cuda") * 8, torch.ones(40, dtype=torch.int32, device="cuda")
    nobody = torch.full((40,), -1, dtype=torch.int32, device="cuda")
    some = torch.where(torch.arange(40, device="cuda") % 4 == 0, -1, torch.arange(40, device="cuda") % 3).to(torch.int32)

    def attend(index):
        return attention(x, r, PagedKVCache(40, 8, 2, 32, dtype=dtype), slots, table, lens, index=index)[0]

    for call in (attend, lambda index: forward(x, r, index=index)[0]):
        want = call(None)
        assert torch.equal(call(nobody), want)
        assert torch.equal(call(some)[some < 0], want[some < 0])
        assert not torch.equal(call(some)[some >= 0], want[some >= 0])
