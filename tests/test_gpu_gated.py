"""The gated activation to 8 bits: bit for bit the quantize kernels' where the activation is exact (relu), within the
activations' own rounding elsewhere."""

from __future__ import annotations

import math

import pytest
import torch

from tricast_b200 import as_operand, gated_quantize, gemm, get_preset, get_scheme, quantize
from tricast_b200.operand import expand_scale

pytestmark = pytest.mark.gpu

SCHEMES = ["fp8_row", "int8_row", "fp8_group128", "mxfp8_e4m3", "mxfp8_e5m2"]
DTYPES = [torch.bfloat16, torch.float16, torch.float32]
SIZES = [(1, 1), (1, 12288), (2, 33), (3, 64), (5, 1000), (7, 1537), (4, 4096), (3, 8200), (2, 16384), (2, 16392), (2, 20001),
         (129, 160), (1500, 96)]


def spec_of(name):
    if name.startswith("group"):
        return get_scheme("fp8_group128").with_(group_size=int(name[5:]))
    return get_scheme(name)


def halves(rows, K, dtype, seed=0, scale=1.5):
    g = torch.Generator(device="cuda").manual_seed(seed + rows * K)
    both = torch.randn(rows, 2 * K, generator=g, device="cuda") * scale
    both[:, :: 61] *= 6
    both = both.to(dtype)
    return both[:, :K], both[:, K:]


def same(q, want):
    assert q.shape == want.shape and q.values.dtype.itemsize == 1
    a, b = q.values.float(), want.values.float()
    if q.values.dtype == torch.int8:  # holds no NaN: its scale, compared below, says so
        b = torch.where(b != b, 0.0, b)
        a = torch.where((b == 0) & torch.isnan(expand_scale(q.scale, q.spec, *a.shape)), 0.0, a)
    assert torch.equal(a.nan_to_num(9e9), b.nan_to_num(9e9))
    if q.values.dtype != torch.int8:  # int8 has one zero
        assert torch.equal(torch.signbit(a) & (a == a), torch.signbit(b) & (b == b))
    assert torch.equal(q.scale.float().nan_to_num(9e9), want.scale.float().nan_to_num(9e9))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("scheme", [*SCHEMES, "group16", "group48", "group256"])
@pytest.mark.parametrize("rows, K", SIZES)
def test_relu_is_the_quantized_product(rows, K, scheme, dtype):
    gate, up = halves(rows, K, dtype)
    y = torch.where(gate.float() > 0, gate.float(), 0.0) * up.float()
    same(gated_quantize(gate, up, spec_of(scheme), activation="relu"), quantize(y, spec_of(scheme)))


def formula(g, name):
    if name == "silu":
        return g * torch.special.expit(g)
    if name == "gelu":
        return g * torch.special.ndtr(g)
    if name == "gelu_tanh":
        return g * torch.special.expit(2 * math.sqrt(2 / math.pi) * (g + 0.044715 * g ** 3))
    return g.clamp(min=0)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("scheme", SCHEMES)
@pytest.mark.parametrize("activation", ["silu", "gelu", "gelu_tanh"])
@pytest.mark.parametrize("rows, K", [(1, 4096), (3, 1537), (40, 512), (2, 17000)])
def test_activations(rows, K, activation, scheme, dtype):
    """e = 2**-24, half a step of fp32. Exponentials and erfc are good to 4 steps, the rest of the chain to half a step each; rounded
    arguments change silu, gelu and gelu_tanh by at most 2 e |g|: y is off by at most 16 e |y| + 2 e |g up|. A scale
    follows its domain's largest y (as many e's, and its own division's), and a code is off by half a step of its grid at most."""
    gate, up = halves(rows, K, dtype, seed=5, scale=3.0)
    q = gated_quantize(gate, up, scheme, activation=activation)
    spec = get_scheme(scheme)
    g, u = gate.double(), up.double()
    y = formula(g, activation) * u
    e = 2.0 ** -24
    off = 16 * e * y.abs() + 2 * e * (g * u).abs()
    n = spec.group_size if spec.granularity == "group" else K
    pad = -K % n

    def domains(t):
        return torch.nn.functional.pad(t, (0, pad)).unflatten(1, (-1, n))

    top, top_off = domains(y).abs().amax(-1), domains(off).amax(-1)
    s = q.scale.double()
    if "mx" in scheme:
        emax = 8 if "e4m3" in scheme else 15
        lo, hi = (torch.frexp(t)[1] - 1 - emax for t in (top - top_off, top + top_off))
        half, got = torch.frexp(s)  # a logarithm may land beside a whole number
        got -= 1
        assert (half == 0.5).all()
        assert ((got == lo) | (got == hi)).all()
    else:
        best = 127.0 if scheme == "int8_row" else 448.0
        assert ((s - top / best).abs() <= top_off / best + 2 * e * top / best).all()
    s = s.repeat_interleave(n, 1)[:, :K] if n != K else s
    v = y / s
    if scheme == "int8_row":
        half, clip = torch.full_like(v, 0.5), 127.0
    else:
        m, low, clip = (2, -14, 57344.0) if "e5m2" in scheme else (3, -6, 448.0)
        _, ex = torch.frexp(v)
        half = torch.ldexp(torch.ones_like(v), (ex - 1).clamp(min=low) - m) / 2
        half = half * (1 + 1e-5) * torch.where(v.abs() > torch.ldexp(torch.ones_like(v), ex - 1) * 1.99, 2.0, 1.0)  # the next binade's
    gap = (q.values.double() - v.clamp(-clip, clip)).abs()
    limit = half + off / s + 4 * e * v.abs()
    worst = (gap / limit).max().item()
    assert worst <= 1.0, worst


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("activation", ["silu", "gelu", "gelu_tanh"])
@pytest.mark.parametrize("scheme, rows, K", [("int8_row", 3000, 4096), ("int8_row", 600, 16392), ("int8_row", 1000, 7781), ("group64", 3000, 4096)])
def test_int8_codes_are_those_of_the_formula_step_by_step(scheme, rows, K, activation, dtype):
    """Every operation of the formula rounded to fp32 by itself, the functions CUDA's: the same operations, so no code and no scale differs."""
    spec = get_scheme("int8_row") if scheme == "int8_row" else get_scheme("int8_row").with_(granularity="group", group_size=64)
    gate, up = halves(rows, K, dtype, seed=9)
    g = gate.float()
    if activation == "silu":
        y = g / (1 + torch.exp(-g))
    elif activation == "gelu":
        y = 0.5 * g * (1 + torch.erf(g * math.sqrt(0.5)))
    else:
        y = 0.5 * g * (1 + torch.tanh(math.sqrt(2 / math.pi) * (g + 0.044715 * g * g * g)))
    same(gated_quantize(gate, up, spec, activation=activation), quantize(y * up.float(), spec))


@pytest.mark.parametrize("scheme", SCHEMES)
@pytest.mark.parametrize("K", [64, 1000, 4096])
def test_rows_that_are_not_finite(K, scheme):
    gate, up = halves(9, K, torch.float32)
    gate, up = gate.clone(), up.clone()
    gate[0], up[1] = 0.0, -0.0
    gate[2, 5], up[3, 7], gate[4, 3], up[5, 2] = float("inf"), float("nan"), float("nan"), float("-inf")
    gate[6], up[6] = 1e30, 1e30
    gate[7] = up[7] = 1e-30
    gate[8] = -abs(gate[8])
    y = torch.where(gate > 0, gate, torch.where(gate != gate, gate, 0.0)) * up
    same(gated_quantize(gate, up, scheme, activation="relu"), quantize(y, scheme))


@pytest.mark.parametrize("activation", ["silu", "gelu", "gelu_tanh"])
def test_far_gates(activation):
    """Gates at which exponentials overflow or vanish."""
    gate = torch.tensor([[-3e38, -1000.0, -104.0, -90.0, -88.0, -30.0, -1e-30, 0.0, 1e-30, 30.0, 88.0, 1000.0, 3e38]], device="cuda")
    q = gated_quantize(gate, torch.full_like(gate, 1e-3), get_scheme("fp8_group128").with_(group_size=1), activation=activation)
    got = q.values.double() * q.scale.double()
    want = formula(gate.double(), activation) * 1e-3
    off = (got - want).abs()
    assert torch.isfinite(got).all() and (off <= 1e-5 * want.abs() + 1e-37).all(), off


def test_the_curve_of_gelu():
    """A group of one element has |y| / 448 as its scale. e = 2**-24. t = 1 / (1 + 0.3 a): 3 e, by at most 2.7 (the polynomial's t p' / p
    at a = 0) 8 e; fit and Horner 3 e, exponential 4 e, its rounded argument a**2 / 2 * 3 e, which times |y| is below e |g|; two products
    and the scale's division 3 e: 18 e |y| + e |g|, and 2**-120 where the exponential is flushed."""
    g = torch.cat([torch.linspace(-14, 14, 400001), -torch.logspace(-30, 1.1, 100000), torch.logspace(-30, 30, 100000)]).cuda()[:, None]
    q = gated_quantize(g, torch.ones_like(g), get_scheme("fp8_group128").with_(group_size=1), activation="gelu")
    got, g = q.scale.double() * 448, g.double()
    want = (g * torch.special.ndtr(g)).abs()
    real = want > 1e-35
    e = 2.0 ** -24
    assert ((got - want).abs() <= 18 * e * want + e * g.abs() + 2.0 ** -120)[real].all()
    ends = torch.tensor([[0.0, -0.0, -5.0, -1e30, 5.0, 1e30, -20.0]], device="cuda")
    q = gated_quantize(ends, torch.ones_like(ends), "fp8_row", activation="gelu").values.float()
    assert torch.signbit(q).tolist() == [[False, True, True, True, False, False, True]]
    for inf, want in ((math.inf, math.inf), (-math.inf, math.nan), (math.nan, math.nan)):
        s = gated_quantize(torch.full((1, 8), inf, device="cuda"), torch.ones(1, 8, device="cuda"), "fp8_row", activation="gelu").scale
        ref = quantize(torch.full((1, 8), want, device="cuda"), "fp8_row").scale
        assert torch.equal(s.nan_to_num(9e9), ref.nan_to_num(9e9))


def test_strides_and_offsets():
    spec = get_scheme("mxfp8_e4m3")
    for dtype in DTYPES:
        for shift in (0, 1, 2, 4, 8):
            wide = torch.randn(6, 3 * 256, device="cuda").to(dtype)
            gate, up = wide[:, shift:shift + 256], wide[:, 300 + shift:556 + shift]
            y = torch.where(gate.float() > 0, gate.float(), 0.0) * up.float()
            same(gated_quantize(gate, up, spec, activation="relu"), quantize(y, spec))
            same(gated_quantize(gate.t().contiguous().t(), up, "fp8_row", activation="relu"), quantize(y, "fp8_row"))
    x = torch.randn(2, 3, 128, device="cuda")
    q = gated_quantize(x, x, "fp8_row", activation="relu")
    assert q.shape == (2, 3, 128) and q.values.shape == (6, 128)
    one = x[0, :1]
    q = gated_quantize(one.expand(3, 128), one.expand(3, 128), "fp8_row", activation="relu")
    assert torch.equal(q.values[0].float(), q.values[2].float())


def test_the_operand_of_a_gemm():
    gate, up = halves(33, 256, torch.bfloat16)
    w = quantize(torch.randn(64, 256, device="cuda"), "fp8_row")
    spec = get_preset("nvidia_hopper_fp8").with_(out_format="fp32")
    q = gated_quantize(gate, up, "fp8_row", activation="relu")
    y = torch.where(gate.float() > 0, gate.float(), 0.0) * up.float()
    want = gemm(as_operand(quantize(y, "fp8_row")), as_operand(w), spec)
    assert torch.equal(gemm(q, w, spec), want)


def test_streams_and_graphs():
    gate, up = halves(40, 512, torch.float32)
    gate, up = gate.clone(), up.clone()
    want = gated_quantize(gate, up, "fp8_row")
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        got = gated_quantize(gate, up, "fp8_row")
    stream.synchronize()
    assert torch.equal(got.values.float(), want.values.float())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = gated_quantize(gate, up, "fp8_row")
    gate.copy_(gate.flip(0))
    up.copy_(up.flip(0))
    graph.replay()
    assert torch.equal(got.values.float(), want.values.float().flip(0)) and torch.equal(got.scale, want.scale.flip(0))


def test_refusals():
    gate, up = halves(4, 64, torch.bfloat16)
    for bad in (dict(up=up[:3]), dict(up=up.float()), dict(up=up.cpu()), dict(gate=gate[:0], up=up[:0]), dict(activation="tanh"),
                dict(gate=gate.double(), up=up.double())):
        with pytest.raises(ValueError):
            gated_quantize(**(dict(gate=gate, up=up, spec="fp8_row") | bad))
    for scheme in ("mxfp4", "nvfp4", "fp8_tensor", "fp8_block128"):
        with pytest.raises(NotImplementedError):
            gated_quantize(gate, up, scheme)
