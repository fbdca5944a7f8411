"""RMS norm with residual and an 8-bit output: against the formula in 64 bits, and bit for bit against the
quantize kernels where the norm itself is exact.

Tolerances, fixed by the arithmetic: the sum of squares is a chain of at most K / 256 + 16 fp32 additions
and products of positive terms (relative error below that many half ulps of 2**-24), halved by the square
root, and six further roundings; codes may differ from the rounding of the exact value by half a grid step
plus that error."""

from __future__ import annotations

import pytest
import torch

from tricast_b200 import as_operand, quantize_into, rms_norm_quantize
from tricast_b200.spec import SCHEMES, QuantSpec, ScaleSpec

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.bfloat16, torch.float16]
EPS = 1e-6


def _inputs(rows, k, dtype, seed, residual=True):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, k, generator=g)
    x[:, torch.randperm(k, generator=g)[: max(1, k // 64)]] *= 8
    r = torch.randn(rows, k, generator=g) * 3 if residual else None
    w = 1 + 0.1 * torch.randn(k, generator=g)
    return x.to(dtype).cuda(), None if r is None else r.to(dtype).cuda(), w.to(dtype).cuda()


def _bound(k):
    return (k / 256 + 16) / 2 * 2.0 ** -24 + 6 * 2.0 ** -24


def _norm64(x, r, w, eps=EPS):
    h = x.double() + (0 if r is None else r.double())
    y = h / (h.square().mean(-1, keepdim=True) + eps).sqrt()
    return y if w is None else y * w.double()


def _check(q, spec, y64):
    """Scales and codes of ``q`` against the exact ``y64``."""
    rows, k = y64.shape
    f, tol = spec.format, _bound(k)
    width = spec.group_size if spec.granularity == "group" else k
    top = torch.stack([p.abs().amax(1) for p in y64.split(width, 1)], 1)
    s = q.scale.double()
    assert s.shape == top.shape
    zero = top == 0  # an all-zero domain has a scale of its own
    assert (s[zero] == (2.0 ** -127 if spec.scale.format.kind == "pow2" else 1.0)).all()
    if spec.scale.format.kind == "pow2":
        ratio = top / s / 2.0 ** spec.emax_elem
        assert ((ratio >= 1 - tol) & (ratio < 2 * (1 + tol)) | zero).all()
    else:
        assert ((s * f.max_normal / top - 1).abs() <= tol)[~zero].all()
    v = y64 / s.repeat_interleave(width, 1)[:, :k]
    got = q.values.double()
    if f.kind == "int":
        step = torch.ones_like(v)
    else:
        _, e = torch.frexp(torch.maximum(v.abs(), got.abs()))
        step = torch.ldexp(torch.ones_like(v), (e - 1).clamp(min=f.emin) - f.mbits)
    v = v.clamp(-f.max_normal, f.max_normal)
    assert ((got - v).abs() <= 0.5 * step + v.abs() * 2 * tol).all()


@pytest.mark.parametrize("scheme", ["fp8_row", "int8_row", "fp8_group128", "mxfp8_e4m3", "mxfp8_e5m2"])
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("rows,k", [(1, 1), (1, 31), (3, 64), (5, 100), (2, 4093), (33, 1024), (7, 4096), (2, 16384), (1, 40000)])
def test_against_64_bits(scheme, dtype, rows, k):
    spec = SCHEMES[scheme]
    x, r, w = _inputs(rows, k, dtype, rows + k)
    q, h = rms_norm_quantize(x, w, spec, residual=r, eps=EPS)
    assert torch.equal(h, (x.float() + r.float()).to(dtype))
    assert q.shape == (rows, k) and q.values.dtype.itemsize == 1
    _check(q, spec, _norm64(x, r, w))
    q0, none = rms_norm_quantize(x, w, scheme, eps=EPS)
    assert none is None
    _check(q0, spec, _norm64(x, None, w))


@pytest.mark.parametrize("group", [1, 16, 48, 64, 256, 1000])
def test_group_sizes(group):
    spec = QuantSpec("fp8_e4m3", "group", group_size=group)
    x, r, w = _inputs(9, 736, torch.bfloat16, group)
    q, _ = rms_norm_quantize(x, w, spec, residual=r, eps=EPS)
    _check(q, spec, _norm64(x, r, w))


@pytest.mark.parametrize("scheme", ["fp8_row", "int8_row", "fp8_group128", "mxfp8_e4m3", "mxfp8_e5m2"])
@pytest.mark.parametrize("k", [1, 32, 96, 333, 4096, 8192])
def test_codes_are_those_of_quantize(scheme, k):
    """With x = +-1 and eps = 0 the norm is exact, so y = +-weight in fp32: its codes and scales are the
    quantize kernels', zeros, subnormals, infinities and NaN among the weights included."""
    spec = SCHEMES[scheme]
    g = torch.Generator().manual_seed(k)
    x = (torch.randint(0, 2, (4, k), generator=g) * 2.0 - 1).cuda()
    for case in range(6):
        w = torch.randn(k, generator=g) * 10.0 ** (case - 3)
        if case == 1:
            w[torch.rand(k, generator=g) < 0.9] = 0
        if case == 2:
            w *= 2.0 ** -130
        if case == 3:
            w = torch.ldexp(torch.ones(k), torch.randint(-20, 20, (k,), generator=g))
        if case == 4:
            w[-1] = float("inf")
        if case == 5:
            w[k // 2] = float("nan")
        w = w.cuda()
        q, _ = rms_norm_quantize(x, w, spec, eps=0.0)
        want, _ = quantize_into(x * w, spec)
        assert torch.equal(q.scale.float().view(torch.int32) & 0x7FFFFFFF, want.scale.view(torch.int32) & 0x7FFFFFFF) or \
            torch.equal(torch.nan_to_num(q.scale.float(), nan=-1.0), torch.nan_to_num(want.scale, nan=-1.0))
        got, ref = q.values.float(), want.values.float()
        if spec.format.kind == "int":
            ref = torch.nan_to_num(ref, nan=0.0)  # integer codes have no NaN; the scale carries it
        assert torch.equal(torch.nan_to_num(got, nan=1e9), torch.nan_to_num(ref, nan=1e9))


def test_empty_rows_zeros_and_large_values():
    x = torch.zeros(3, 512, device="cuda", dtype=torch.bfloat16)
    x[1, 7] = 3e38  # its square overflows fp32: the norm of the row is 0, as the formula in fp32 has it
    x[2] = float("nan")
    q, _ = rms_norm_quantize(x, None, "fp8_row", eps=EPS)
    assert (q.values[0].float() == 0).all() and q.scale[0].item() == 1.0
    assert (q.values[1].float() == 0).all()
    assert q.scale[2].isnan().all()


def test_strides_and_leading_dimensions():
    g = torch.Generator().manual_seed(3)
    wide = torch.randn(2, 9, 1000, generator=g).bfloat16().cuda()
    w = torch.rand(333, generator=g).cuda()
    for x in (wide[..., 1:334], wide[..., 8:341], wide[:, :, 0:999:3], wide[:, ::2, 5:338]):
        r = torch.flip(x, (0,))
        q, h = rms_norm_quantize(x, w, "fp8_row", residual=r)
        c, hc = rms_norm_quantize(x.contiguous(), w, "fp8_row", residual=r.contiguous())
        assert q.shape == tuple(x.shape) and torch.equal(h, hc)
        assert torch.equal(q.values.view(torch.uint8), c.values.view(torch.uint8)) and torch.equal(q.scale, c.scale)


def test_another_stream_and_repeated_calls_agree():
    x, r, w = _inputs(257, 5120, torch.bfloat16, 1)
    first, h = rms_norm_quantize(x, w, "mxfp8_e4m3", residual=r)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        second, h2 = rms_norm_quantize(x, w, "mxfp8_e4m3", residual=r)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(first.values.view(torch.uint8), second.values.view(torch.uint8)) and torch.equal(h, h2)
    assert torch.equal(first.scale.view(torch.uint8), second.scale.view(torch.uint8))


@pytest.mark.parametrize("scheme", ["fp8_row", "int8_row", "mxfp8_e4m3"])
def test_the_result_is_a_gemm_operand(scheme):
    from tricast_b200 import gemm
    from tricast_b200.spec import MMASpec

    x, r, w = _inputs(24, 256, torch.bfloat16, 2)
    q, _ = rms_norm_quantize(x, w, scheme, residual=r)
    weight, _ = quantize_into(torch.randn(40, 256, generator=torch.Generator().manual_seed(4)).cuda(), SCHEMES[scheme])
    out = gemm(q, weight, MMASpec("fp64", out_format="fp32"))
    want = q.dequantize().double() @ weight.dequantize().double().T
    # One fp32 rounding of each scaled operand value and of the result.
    size = q.dequantize().double().abs() @ weight.dequantize().double().abs().T
    assert ((out.double() - want).abs() <= size * 2.0 ** -21).all()
    op = as_operand(q)
    assert op.scale.dtype == torch.float32


def test_refusals():
    x = torch.zeros(4, 64, device="cuda")
    w = torch.ones(64, device="cuda")
    with pytest.raises(ValueError, match="CUDA tensor"):
        rms_norm_quantize(x.cpu(), w.cpu(), "fp8_row")
    with pytest.raises(ValueError, match="nonempty"):
        rms_norm_quantize(x[:0], w, "fp8_row")
    with pytest.raises(ValueError, match="residual"):
        rms_norm_quantize(x, w, "fp8_row", residual=x.bfloat16())
    with pytest.raises(ValueError, match="weight"):
        rms_norm_quantize(x, w[:32], "fp8_row")
    with pytest.raises(ValueError, match="eps"):
        rms_norm_quantize(x, w, "fp8_row", eps=-1.0)
    with pytest.raises(ValueError, match="dtype"):
        rms_norm_quantize(x.double(), w, "fp8_row")
    with pytest.raises(ValueError, match="unknown scheme"):
        rms_norm_quantize(x, w, "fp9_row")
    for spec in (SCHEMES["mxfp4"], SCHEMES["nvfp4"], SCHEMES["fp8_tensor"], SCHEMES["fp8_block128"], SCHEMES["bf16"],
                 SCHEMES["int4_g128_zp"], QuantSpec("fp8_e4m3", "row", rounding="rtz"),
                 QuantSpec("fp8_e4m3", "row", scale=ScaleSpec("fp16"))):
        with pytest.raises(NotImplementedError):
            rms_norm_quantize(x, w, spec)
