"""What the norm returns as a GEMM operand: groups of 128 and E5M2 elements against the product in 64 bits, and the
class that a spec of TriCast's own asks for."""

from __future__ import annotations

import dataclasses
import sys
import types

import pytest
import torch

from tricast_b200 import gemm, quantize_into, rms_norm_quantize
from tricast_b200.formats import container_dtype
from tricast_b200.operand import QTensor
from tricast_b200.spec import SCHEMES, MMASpec, QuantSpec

pytestmark = pytest.mark.gpu


def _inputs(rows, k, seed):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, k, generator=g)
    return x.bfloat16().cuda(), (torch.randn(rows, k, generator=g) * 3).bfloat16().cuda(), torch.rand(k, generator=g).bfloat16().cuda()


@pytest.mark.parametrize("spec", [SCHEMES["fp8_group128"], SCHEMES["mxfp8_e5m2"], QuantSpec("fp8_e5m2", "row")],
                         ids=["fp8_group128", "mxfp8_e5m2", "fp8_e5m2_row"])
@pytest.mark.parametrize("k", [256, 512])
def test_groups_and_e5m2(spec, k):
    x, r, w = _inputs(24, k, k)
    q, _ = rms_norm_quantize(x, w, spec, residual=r)
    weight, _ = quantize_into(torch.randn(40, k, generator=torch.Generator().manual_seed(4)).cuda(), spec)
    out = gemm(q, weight, MMASpec("fp64", out_format="fp32"))
    want = q.dequantize().double() @ weight.dequantize().double().T
    # One fp32 rounding of each scaled operand value and of the result.
    size = q.dequantize().double().abs() @ weight.dequantize().double().abs().T
    assert ((out.double() - want).abs() <= size * 2.0 ** -21).all()


@pytest.mark.parametrize("scheme", ["fp8_row", "mxfp8_e4m3", "int8_row"])
def test_a_tricast_spec_gets_tricasts_class(scheme, monkeypatch):
    """As ``quantize`` has it: values in the format's container, scales in fp32."""

    class Theirs(QTensor):
        pass

    for name in ("tricast", "tricast.quant", "tricast.quant.qtensor"):
        monkeypatch.setitem(sys.modules, name, types.ModuleType(name))
    sys.modules["tricast.quant.qtensor"].QTensor = Theirs
    spec = SCHEMES[scheme]
    foreign = type("TheirSpec", (type(spec),), {"__module__": "tricast.spec"})
    theirs = foreign(**{f.name: getattr(spec, f.name) for f in dataclasses.fields(spec) if f.init})
    x, r, w = _inputs(9, 128, 1)
    q, h = rms_norm_quantize(x, w, theirs, residual=r)
    ours, same = rms_norm_quantize(x, w, spec, residual=r)
    assert type(q) is Theirs and q.spec is theirs and q.shape == (9, 128)
    assert q.values.dtype == container_dtype(spec.format) and q.scale.dtype == torch.float32
    assert torch.equal(q.dequantize(), ours.dequantize()) and torch.equal(h, same)
    assert torch.equal(quantize_into(x, theirs)[0].values, quantize_into(x, spec)[0].values)
