"""Low-rank adapters of many requests beside a shared projection. No TriCast counterpart."""

from __future__ import annotations

import torch

from . import _native as N

_CODES = {torch.float8_e4m3fn: 3, torch.float8_e5m2: 4, torch.int8: 5}


def low_rank_add(y: torch.Tensor, x, a: torch.Tensor, b: torch.Tensor, index: torch.Tensor, *, gain: torch.Tensor | None = None,
                 dtype: torch.dtype | None = None) -> torch.Tensor:
    """``y + gain[i] * (x a[i]^T) b[i]^T`` for each token, ``i = index[token]`` its adapter.

    ``y`` ``[tokens, n]``: the shared projection of ``x``, as :func:`gemm` gives it or in 16 bits. ``x`` ``[tokens, k]``: a
    tensor, or the QTensor that the projection read (8-bit or container values with one fp32 scale a row, as
    :func:`rms_norm_quantize` and :func:`quantize` give them for ``fp8_row`` and ``int8_row``). ``a`` ``[adapters, rank, k]``
    and ``b`` ``[adapters, n, rank]`` (contiguous; ranks below the pool's are padded with zeros), ``index`` int32 ``[tokens]``: an
    index outside the pool (``-1``) adds nothing. ``gain`` fp32 ``[adapters]``: a factor of each adapter.

    The sums are fp32, rounded once to ``dtype`` (default ``y``'s). Weights of 16 bits with ``x`` of their type or 8-bit
    codes, ``y`` and ``dtype`` of their type or fp32, and ranks up to 128 go through the tensor cores, anything else element
    by element. On the tensor cores the first product enters the second one in parts of the weights' type: two where
    ``dtype`` has 16 bits (2**-16 of it is left out in bf16, 2**-22 in fp16), three where it has 32 (2**-24, as fp32
    itself). An infinite ``x`` or weight of ``a`` gives what fp32 does; one of ``b``, which its column's tokens alone see,
    may give NaN in place of an infinity. What a token gets depends on no other token's values or adapter, to the bit, but
    sums are cut by how many tokens there are. Any order of tokens is allowed; those of one adapter that stand together
    share its weights' way through the chip. More than some 250 tokens take scratch memory (up to 6 bytes a token and rank)
    while they run. No gradients pass: the output is detached."""
    if not y.is_cuda:
        raise ValueError("the B200 backend requires a CUDA tensor")
    device, scale = y.device, None
    if not isinstance(x, torch.Tensor):
        spec = x.spec
        if spec.granularity != "row" or x.scale is None or x.zero_point is not None or x.global_scale is not None:
            raise NotImplementedError("low_rank_add takes a QTensor with one scale a row")
        x, scale = x.values, x.scale
        if scale.dtype != torch.float32 or scale.numel() != x.shape[0] or not scale.is_contiguous() or scale.device != device:
            raise NotImplementedError("low_rank_add takes a QTensor with one fp32 scale a row on y's device")
    if y.ndim != 2 or x.ndim != 2 or x.shape[0] != y.shape[0] or x.device != device:
        raise ValueError("y must be [tokens, n] and x [tokens, k] on one device")
    tokens, n = y.shape
    k = x.shape[1]
    if a.ndim != 3 or b.ndim != 3 or a.shape[2] != k or b.shape != (a.shape[0], n, a.shape[1]) or a.dtype != b.dtype:
        raise ValueError("a must be [adapters, rank, k] and b [adapters, n, rank] of one dtype")
    if a.device != device or b.device != device or not a.is_contiguous() or not b.is_contiguous():
        raise ValueError("a and b must be contiguous, on y's device")
    if index.shape != (tokens,) or index.dtype != torch.int32 or index.device != device:
        raise ValueError("index must be an int32 tensor [tokens] on y's device")
    if gain is not None and (gain.shape != a.shape[:1] or gain.dtype != torch.float32 or gain.device != device):
        raise ValueError("gain must be an fp32 tensor [adapters] on y's device")
    kind = _CODES.get(x.dtype)
    if kind is None:
        kind = N.dtype_code(x.dtype)
    elif scale is None:
        raise ValueError("8-bit codes need a QTensor with their scales")
    dtype = dtype or y.dtype
    y_code, w_code, out_code = N.dtype_code(y.dtype), N.dtype_code(a.dtype), N.dtype_code(dtype)
    if x.stride(1) != 1 or x.stride(0) < k:
        x = x.contiguous()
    if y.stride(1) != 1 or y.stride(0) < n:
        y = y.contiguous()
    if index.stride(0) != 1:
        index = index.contiguous()
    if gain is not None and gain.stride(0) != 1:
        gain = gain.contiguous()
    out = torch.empty((tokens, n), dtype=dtype, device=device)
    at = device.index
    lib, rank = N.lib(), a.shape[1]
    with N.on_device(at):
        nbytes = lib.tc_low_rank_add_workspace(tokens, kind, w_code, rank, y_code, out_code)
        ws = torch.empty(nbytes, dtype=torch.uint8, device=device) if nbytes else None
        status = lib.tc_low_rank_add(
            y.data_ptr(), y_code, max(y.stride(0), n), x.data_ptr(), kind, max(x.stride(0), k),
            None if scale is None else scale.data_ptr(), tokens, k, n, a.data_ptr(), b.data_ptr(), w_code, a.shape[0], rank,
            None if gain is None else gain.data_ptr(), index.data_ptr(), out.data_ptr(), out_code,
            None if ws is None else ws.data_ptr(), nbytes, N.raw_stream(at))
    if status:
        N.check(status, "tc_low_rank_add")
    return out


__all__ = ["low_rank_add"]
