"""INT8 codes of the gated activation where gates are tiny or large: every division is the formula's."""

from __future__ import annotations

import math

import pytest
import torch

from tricast_b200 import gated_quantize, get_scheme, quantize

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("activation", ["silu", "gelu", "gelu_tanh"])
@pytest.mark.parametrize("group", [0, 64])
def test_gates_of_every_magnitude(activation, group):
    """A row of gates for each power of two from the least subnormal to 2**6, with ups that bring them up to where they can be:
    each step of the formula rounded by itself gives the same codes and scales."""
    g = torch.Generator(device="cuda").manual_seed(1)
    e = torch.arange(-149, 7, device="cuda")[:, None]
    shape = (e.shape[0], 2048)
    gate = torch.ldexp((1 + torch.rand(shape, generator=g, device="cuda")).double(), e).float()
    gate = torch.where(torch.rand(shape, generator=g, device="cuda") < 0.5, -gate, gate)
    up = (torch.ldexp(torch.randn(shape, generator=g, device="cuda").double(), (-e).clamp(max=120))).float()
    if activation == "silu":
        y = gate / (1 + torch.exp(-gate))
    elif activation == "gelu":
        y = 0.5 * gate * (1 + torch.erf(gate * math.sqrt(0.5)))
    else:
        y = 0.5 * gate * (1 + torch.tanh(math.sqrt(2 / math.pi) * (gate + 0.044715 * gate * gate * gate)))
    spec = get_scheme("int8_row")
    if group:
        spec = spec.with_(granularity="group", group_size=group)
    q, want = gated_quantize(gate, up, spec, activation=activation), quantize(y * up, spec)
    assert torch.equal(q.scale, want.scale)
    assert torch.equal(q.values.float(), want.values.float())
