"""Root-mean-square norm with the residual's addition and an output in 8 bits with scales: what stands
between a layer's residual stream and a quantized GEMM operand. No TriCast counterpart (TriCast quantizes
the norm's output in a pass of its own, ``src/tricast/nn/linear.py:342-350``)."""

from __future__ import annotations

import torch

from . import _native as N
from .formats import container_dtype
from .operand import QTensor, qtensor_class
from .quantize import _qspec

_CODE_DTYPES = {("float", 4): torch.float8_e4m3fn, ("float", 5): torch.float8_e5m2}
_PREPARED: dict = {}  # spec object -> (it, its C descriptor, code dtype, group size, scale dtype, class of the result)


def _prepared(spec):
    hit = _PREPARED.get(id(spec))
    if hit is None or hit[0] is not spec:
        if getattr(spec, "scale", None) is None:
            raise NotImplementedError("rms_norm_quantize needs a spec with scales")
        f = spec.format
        code = torch.int8 if f.kind == "int" else _CODE_DTYPES.get((f.kind, getattr(f, "ebits", 0)), torch.uint8)
        group = spec.group_size if spec.granularity == "group" else 0
        if len(_PREPARED) >= 64:
            _PREPARED.clear()
        hit = _PREPARED[id(spec)] = (
            spec, _qspec(spec), code, group, torch.float8_e8m0fnu if spec.scale.format.kind == "pow2" else torch.float32,
            qtensor_class(spec))
    return hit


def _rows(x: torch.Tensor, K: int) -> tuple:
    """``x`` as rows of K contiguous elements, and their stride."""
    if x.ndim != 2:
        x = x.reshape(-1, K)
    step, one = x.stride()
    if (one != 1 and K > 1) or step < K:
        x = x.contiguous()
        step = K
    return x, step


def rms_norm_quantize(x: torch.Tensor, weight: torch.Tensor | None, spec, *, residual: torch.Tensor | None = None,
                      eps: float = 1e-6):
    """``(QTensor, h)``: the quantized ``h / sqrt(mean(h**2) + eps) * weight`` over the last dimension, with
    ``h = x + residual``, and ``h`` in ``x``'s dtype (``None`` without a residual).

    ``spec``: a scheme name or spec with 8-bit elements (``fp8_e4m3``, ``fp8_e5m2``, ``int8``), row or group
    granularity and fp32 absmax or E8M0 scales (``fp8_row``, ``int8_row``, ``fp8_group128``, ``mxfp8_*``).
    The QTensor's values are held in the 8-bit torch dtype of the format and E8M0 scales in
    ``torch.float8_e8m0fnu``; it is an operand of :func:`gemm` like any other (with a spec of TriCast's own it is
    TriCast's class, as :func:`quantize` returns it). The norm is computed in fp32 from the unrounded ``h``, and codes
    and scales are those :func:`quantize` gives for the fp32 result. No gradients pass: both outputs are detached."""
    if isinstance(spec, str):
        from .spec import get_scheme

        spec = get_scheme(spec)
    _, qs, code_dtype, group, scale_dtype, cls = _prepared(spec)
    if not x.is_cuda:
        raise ValueError("the B200 backend requires a CUDA tensor")
    shape = x.shape
    if not shape or x.numel() == 0:
        raise ValueError("rms_norm_quantize needs a nonempty tensor of shape [..., K]")
    dtype = N.dtype_code(x.dtype)
    K = shape[-1]
    device = x.device
    x2, stride = _rows(x, K)
    r2, rstride = None, K
    if residual is not None:
        if residual.shape != shape or residual.dtype != x.dtype or residual.device != device:
            raise ValueError("residual must have x's shape, dtype and device")
        r2, rstride = _rows(residual, K)
    wdt = 0
    if weight is not None:
        if weight.shape != (K,) or weight.device != device:
            raise ValueError("weight must have shape [K] on x's device")
        wdt = N.dtype_code(weight.dtype)
        if weight.stride(0) != 1:
            weight = weight.contiguous()
    rows = x2.shape[0]
    values = torch.empty((rows, K), device=device, dtype=code_dtype)
    scale = torch.empty((rows, -(-K // group) if group else 1), device=device, dtype=scale_dtype)
    h = None if r2 is None else torch.empty(shape, device=device, dtype=x.dtype)
    index = device.index
    with N.on_device(index):
        status = N.lib().tc_rms_norm_quantize(
            x2.data_ptr(), None if r2 is None else r2.data_ptr(), dtype, rows, K, stride, rstride,
            None if weight is None else weight.data_ptr(), wdt, eps, qs, values.data_ptr(), scale.data_ptr(),
            None if h is None else h.data_ptr(), N.raw_stream(index))
    if status:
        N.check(status, "tc_rms_norm_quantize")
    if cls is not QTensor:  # TriCast's holds values in the format's container and scales in fp32
        values, scale = values.to(container_dtype(spec.format)), scale.to(torch.float32)
    return cls(values, scale, None, None, spec, tuple(shape)), h


__all__ = ["rms_norm_quantize"]
