"""Gated activation with an output in 8 bits with scales: what stands between the two GEMMs of a feed-forward block, as
:func:`rms_norm_quantize` stands before the first. No TriCast counterpart (TriCast quantizes the product in a pass of its own,
``src/tricast/nn/linear.py:342-350``)."""

from __future__ import annotations

import torch

from . import _native as N
from .formats import container_dtype
from .norm import _prepared, _rows
from .operand import QTensor

ACTIVATION_CODES = {"silu": 0, "gelu": 1, "gelu_tanh": 2, "relu": 3}


def gated_quantize(gate: torch.Tensor, up: torch.Tensor, spec, *, activation: str = "silu"):
    """QTensor of ``activation(gate) * up`` over the last dimension.

    ``gate`` and ``up`` ``[..., K]`` (any row strides: two halves of one projection's output, say); ``activation``: ``"silu"``,
    ``"gelu"``, ``"gelu_tanh"`` or ``"relu"``. ``spec`` as for :func:`rms_norm_quantize` (8-bit elements, row or group
    granularity, fp32 absmax or E8M0 scales), and so is the QTensor. The product is fp32, and codes and scales are those
    :func:`quantize` gives for it. For INT8 codes it is that of PyTorch's operations one by one; for the others the activation's
    exponential and reciprocal are the hardware's, which is mostly nearer to the formula (2 halves of an fp32 step of ``gate * up``, 16 of
    the product) but not PyTorch's to the bit: a code may be the neighbouring one where the quotient lies that near the middle between two
    (one in some 10**5 or 10**6), a power-of-two scale where the maximum lies that near a power of two (one in some 10**8). No gradients
    pass: the output is detached."""
    if isinstance(spec, str):
        from .spec import get_scheme

        spec = get_scheme(spec)
    _, qs, code_dtype, group, scale_dtype, cls = _prepared(spec, "gated_quantize")
    if activation not in ACTIVATION_CODES:
        raise ValueError(f"unknown activation {activation!r}; known: {list(ACTIVATION_CODES)}")
    if not gate.is_cuda:
        raise ValueError("the B200 backend requires a CUDA tensor")
    shape, device = gate.shape, gate.device
    if not shape or gate.numel() == 0:
        raise ValueError("gated_quantize needs nonempty tensors of shape [..., K]")
    if up.shape != shape or up.dtype != gate.dtype or up.device != device:
        raise ValueError("up must have gate's shape, dtype and device")
    dtype = N.dtype_code(gate.dtype)
    K = shape[-1]
    (g2, g_stride), (u2, u_stride) = _rows(gate, K), _rows(up, K)
    rows = g2.shape[0]
    values = torch.empty((rows, K), device=device, dtype=code_dtype)
    scale = torch.empty((rows, -(-K // group) if group else 1), device=device, dtype=scale_dtype)
    index = device.index
    with N.on_device(index):
        status = N.lib().tc_gated_quantize(g2.data_ptr(), g_stride, u2.data_ptr(), u_stride, dtype, rows, K,
                                           ACTIVATION_CODES[activation], qs, values.data_ptr(), scale.data_ptr(),
                                           N.raw_stream(index))
    if status:
        N.check(status, "tc_gated_quantize")
    if cls is not QTensor:  # TriCast's holds values in the format's container and scales in fp32
        values, scale = values.to(container_dtype(spec.format)), scale.to(torch.float32)
    return cls(values, scale, None, None, spec, tuple(shape))


__all__ = ["gated_quantize"]
