"""Paged key / value cache, quantized as it is written (TriCast emulates a quantized cache on the host side,
``src/tricast/kv/``; this one holds the codes)."""

from __future__ import annotations

import ctypes as C

import torch

from . import _native as N

_CODES = {"fp8_row": torch.float8_e4m3fn, "int8_row": torch.int8, "mxfp4": torch.uint8}


class PagedKVCache:
    """``num_pages`` pages of ``page_size`` tokens for ``kv_heads`` heads of ``head_dim`` elements.

    ``scheme``: ``"fp8_row"`` (E4M3 codes) or ``"int8_row"``, with one fp32 absmax scale per token and head;
    ``"mxfp4"`` (E2M1 codes, two a byte, and one E8M0 scale per 32 elements); ``None`` (as they come).
    ``dtype``: of the keys, values and queries. Slot ``s`` is token ``s % page_size`` of page
    ``s // page_size``; which pages a sequence owns is the caller's to keep.

    ``k`` and ``v`` hold the codes ``[num_pages, kv_heads, page_size, head_dim]`` (``mxfp4``: ``head_dim / 2``
    bytes), ``k_scale`` and ``v_scale`` the scales ``[num_pages, kv_heads, page_size]`` (``mxfp4``:
    ``[..., head_dim / 32]``); they may be copied and shared but not replaced."""

    def __init__(self, num_pages: int, page_size: int, kv_heads: int, head_dim: int, scheme: str | None = "fp8_row", *,
                 dtype: torch.dtype = torch.bfloat16, device="cuda"):
        if scheme not in N.KV_SCHEME_CODES:
            raise ValueError(f"unknown cache scheme {scheme!r}; known: {list(N.KV_SCHEME_CODES)}")
        code = N.dtype_code(dtype)
        if not 8 <= page_size <= 256 or page_size & (page_size - 1):
            raise ValueError("page_size must be a power of two in [8, 256]")
        if not 16 <= head_dim <= 256 or head_dim % (32 if scheme == "mxfp4" else 16):
            raise ValueError("head_dim must be a multiple of 16 (mxfp4: 32) in [16, 256]")
        if num_pages < 1 or not 1 <= kv_heads <= 65535:
            raise ValueError("num_pages and kv_heads must be positive")
        self.num_pages, self.page_size, self.kv_heads, self.head_dim = num_pages, page_size, kv_heads, head_dim
        self.scheme, self.dtype, self._row = scheme, dtype, (kv_heads, head_dim)
        device = torch.device(device)
        if device.type != "cuda":
            raise ValueError("the B200 backend requires a CUDA device")
        if device.index is None:
            device = torch.device("cuda", torch.cuda.current_device())
        self.device = device
        lead = (num_pages, kv_heads, page_size)
        width = head_dim // 2 if scheme == "mxfp4" else head_dim
        kind = dtype if scheme is None else _CODES[scheme]

        def zeros(shape, kind):
            return torch.zeros((*shape[:-1], shape[-1] * kind.itemsize), dtype=torch.uint8, device=device).view(kind)

        self.k, self.v = zeros((*lead, width), kind), zeros((*lead, width), kind)
        self.k_scale = self.v_scale = None
        if scheme == "mxfp4":
            shape, kind = (*lead, head_dim // 32), torch.float8_e8m0fnu
            self.k_scale, self.v_scale = zeros(shape, kind), zeros(shape, kind)
        elif scheme is not None:
            self.k_scale, self.v_scale = zeros(lead, torch.float32), zeros(lead, torch.float32)
        d = N.TcKvCache()
        d.k, d.v = self.k.data_ptr(), self.v.data_ptr()
        d.k_scale = 0 if self.k_scale is None else self.k_scale.data_ptr()
        d.v_scale = 0 if self.v_scale is None else self.v_scale.data_ptr()
        d.scheme, d.dtype = N.KV_SCHEME_CODES[scheme], code
        d.num_pages, d.page_size, d.kv_heads, d.head_dim = num_pages, page_size, kv_heads, head_dim
        self._desc, self._ref = d, C.byref(d)

    @property
    def capacity(self) -> int:
        """Tokens the cache holds."""
        return self.num_pages * self.page_size

    def _slots(self, slots: torch.Tensor) -> torch.Tensor:
        if slots.ndim != 1 or slots.dtype != torch.int64 or slots.device != self.device:
            raise ValueError("slots must be a 1-D int64 tensor on the cache's device")
        return slots if slots.is_contiguous() else slots.contiguous()

    def _rows(self, x: torch.Tensor, tokens: int, name: str) -> torch.Tensor:
        if x.shape != (tokens, *self._row) or x.dtype != self.dtype or x.device != self.device:
            raise ValueError(f"{name} must be [tokens, {self.kv_heads}, {self.head_dim}] of {self.dtype} on the cache's device")
        return x if x.stride(2) == 1 else x.contiguous()

    def write(self, k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor) -> None:
        """Quantize ``k`` and ``v`` ``[tokens, kv_heads, head_dim]`` into ``slots`` (int64 ``[tokens]``) on the
        current stream. Tokens whose slot is outside the cache (``-1``) are skipped. The other slots must differ: one
        that several tokens name may end with codes of one and scales of another (no other slot is touched)."""
        slots = self._slots(slots)
        tokens = slots.shape[0]
        k, v = self._rows(k, tokens, "k"), self._rows(v, tokens, "v")
        ks, vs, index = k.stride(), v.stride(), self.device.index
        with N.on_device(index):
            status = N.lib().tc_kv_write(self._ref, k.data_ptr(), ks[0], ks[1], v.data_ptr(), vs[0], vs[1],
                                         slots.data_ptr(), tokens, N.raw_stream(index))
        if status:
            N.check(status, "tc_kv_write")

    def read(self, slots: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
        """The keys and values at ``slots``, dequantized to the cache's dtype: ``[tokens, kv_heads, head_dim]``
        each (zeros for a slot outside the cache)."""
        slots = self._slots(slots)
        tokens = slots.shape[0]
        k = torch.empty((tokens, self.kv_heads, self.head_dim), dtype=self.dtype, device=self.device)
        v = torch.empty_like(k)
        index = self.device.index
        with N.on_device(index):
            status = N.lib().tc_kv_read(self._ref, slots.data_ptr(), tokens, k.data_ptr(), v.data_ptr(),
                                        N.raw_stream(index))
        if status:
            N.check(status, "tc_kv_read")
        return k, v


__all__ = ["PagedKVCache"]
