"""The sign of zero in 8-bit float codes: those of the quantize kernels, byte for byte, from every kernel that casts."""

from __future__ import annotations

import pytest
import torch

from tricast_b200 import PagedKVCache, quantize_into, rms_norm_quantize
from tricast_b200.spec import SCHEMES, QuantSpec

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("spec", [SCHEMES["fp8_row"], SCHEMES["fp8_group128"], QuantSpec("fp8_e5m2", "row"),
                                  SCHEMES["mxfp8_e4m3"]], ids=lambda s: f"{s.format.name}-{s.granularity}-{s.group_size}")
@pytest.mark.parametrize("k", [64, 333, 512, 40000])
def test_norm(spec, k):
    """x = +-1 and eps = 0: the norm is exact, and a weight of 0 gives zeros of either sign."""
    g = torch.Generator().manual_seed(k)
    x = (torch.randint(0, 2, (5, k), generator=g) * 2.0 - 1).cuda()
    w = torch.randn(k, generator=g)
    w[torch.rand(k, generator=g) < 0.5] = 0
    for weight in (w.cuda(), torch.zeros(k, device="cuda")):
        q, _ = rms_norm_quantize(x, weight, spec, eps=0.0)
        want, extras = quantize_into(x * weight, spec, want_codes=True)
        assert (extras.codes == 0x80).any()
        assert torch.equal(q.values.view(torch.uint8), extras.codes.view(q.values.shape))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16], ids=str)
@pytest.mark.parametrize("scheme", ["fp8_row", "mxfp4"])
def test_cache(scheme, dtype):
    g = torch.Generator().manual_seed(1)
    x = torch.randn(40, 3, 64, generator=g)
    x[torch.rand(x.shape, generator=g) < 0.4] = -0.0
    x[7] = -0.0
    x = x.to(dtype).cuda()
    cache = PagedKVCache(3, 16, 3, 64, scheme, dtype=dtype)
    slots = torch.arange(40, device="cuda")
    cache.write(x, x, slots)
    _, extras = quantize_into(x.reshape(-1, 64), SCHEMES[scheme], want_codes=True)
    for pool in (cache.k, cache.v):
        got = pool.view(torch.uint8)[slots // 16, :, slots % 16]
        assert torch.equal(got, extras.codes.view(got.shape))
