"""Attention of a chunk of new tokens (a prefill chunk, drafted tokens or a decode step) over a
:class:`PagedKVCache`, reading its codes."""

from __future__ import annotations

import torch

from . import _native as N


def _index(t: torch.Tensor, shape, device, name: str) -> None:
    if t.dtype != torch.int32 or t.device != device or t.shape != shape:
        raise ValueError(f"{name} must be an int32 tensor of shape {list(shape)} on the cache's device")


def paged_attention(q: torch.Tensor, cache, block_table: torch.Tensor, seq_lens: torch.Tensor,
                    cu_q: torch.Tensor | None = None, *, max_q_len: int | None = None, scale: float | None = None,
                    causal: bool = True, window: int = 0, return_lse: bool = False):
    """``softmax(scale * q k^T) v`` of each sequence's last tokens over its cached keys and values.

    ``q`` ``[total_q, heads, head_dim]`` of the cache's dtype (any strides with contiguous elements), query head
    ``h`` reading key / value head ``h // (heads // kv_heads)``. ``cu_q`` (int32 ``[batch + 1]``): sequence ``b``'s
    new tokens are ``q[cu_q[b]:cu_q[b + 1]]``, of which the first ``max_q_len`` are computed (default: ``total_q``; the
    bound also chooses the kernel, so a decode step should give it); without it every sequence has one. ``seq_lens`` (int32 ``[batch]``): the sequence's context, the new tokens, written
    before this call, included. ``block_table`` (int32 ``[batch, max_pages]``): the page of each ``page_size``
    positions; entries past the context are not read, and keys on a page outside the cache (``-1``) count as
    absent. ``causal``: a token sees itself and what precedes it, the last ``window`` positions of that where
    ``window > 0``. ``scale`` defaults to ``1 / sqrt(head_dim)``.

    Returns ``[total_q, heads, head_dim]`` in the cache's dtype, and with ``return_lse`` the fp32 natural
    logarithms of the softmax sums ``[total_q, heads]``. A token that sees no key gives zeros and ``-inf``, as does one
    of no sequence (before ``cu_q[0]``, from ``cu_q[batch]`` on) or beyond ``max_q_len``.
    Chunks of many tokens over a quantized cache take up to 512 MiB of scratch memory while they run. No gradients
    pass: the outputs are detached."""
    device = cache.device
    if q.ndim != 3 or q.shape[2] != cache.head_dim or q.dtype != cache.dtype or q.device != device:
        raise ValueError(f"q must be [tokens, heads, {cache.head_dim}] of {cache.dtype} on the cache's device")
    total, heads, dim = q.shape
    if heads == 0 or heads % cache.kv_heads:
        raise ValueError("the number of query heads must be a multiple of the cache's")
    if block_table.ndim != 2 or block_table.dtype != torch.int32 or block_table.device != device:
        raise ValueError("block_table must be an int32 tensor [batch, max_pages] on the cache's device")
    batch, max_pages = block_table.shape
    _index(seq_lens, (batch,), device, "seq_lens")
    if cu_q is not None:
        _index(cu_q, (batch + 1,), device, "cu_q")
        if cu_q.stride(0) != 1:
            cu_q = cu_q.contiguous()
    elif total != batch:
        raise ValueError("without cu_q every sequence has one new token: q needs as many tokens as block_table rows")
    if window < 0 or (window and not causal):
        raise ValueError("window must be positive and needs causal=True")
    if max_q_len is not None and max_q_len < 1:
        raise ValueError("max_q_len must be positive")
    # Both bounds go on as 32-bit numbers: beyond these they bound nothing (contexts hold at most 2**30 tokens).
    if cu_q is None:
        max_q_len = 1
    elif max_q_len is None or max_q_len > total:
        max_q_len = total or 1
    if window > 1 << 30:
        window = 1 << 30
    if q.stride(2) != 1:
        q = q.contiguous()
    table_stride, one = block_table.stride()
    if one != 1 and max_pages > 1:
        block_table = block_table.contiguous()
        table_stride = max_pages
    if seq_lens.stride(0) != 1:
        seq_lens = seq_lens.contiguous()
    out = torch.empty((total, heads, dim), dtype=q.dtype, device=device)
    lse = torch.empty((total, heads), dtype=torch.float32, device=device) if return_lse else None
    lib = N.lib()
    index = device.index
    token_stride, head_stride, _ = q.stride()
    with N.on_device(index):
        nbytes = lib.tc_paged_attention_workspace(cache._ref, heads, total, batch, max_q_len, max_pages)
        ws = torch.empty(nbytes, dtype=torch.uint8, device=device) if nbytes else None
        status = lib.tc_paged_attention(
            cache._ref, q.data_ptr(), token_stride, head_stride, total, heads, block_table.data_ptr(), table_stride,
            max_pages, seq_lens.data_ptr(), None if cu_q is None else cu_q.data_ptr(), batch, max_q_len,
            dim ** -0.5 if scale is None else scale, causal, window, out.data_ptr(),
            None if lse is None else lse.data_ptr(), None if ws is None else ws.data_ptr(), nbytes,
            N.raw_stream(index))
    if status:
        N.check(status, "tc_paged_attention")
    return (out, lse) if return_lse else out


__all__ = ["paged_attention"]
