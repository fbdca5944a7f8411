"""One attention layer as a server runs it: norm to an 8-bit operand, QKV GEMM, cache write, attention over the cache,
output GEMM, the GEMMs under an emulated accumulation rule (attention's two products run on the tensor cores as they
are). It shows the serving operators together and measures what a cache scheme costs end to end; ``python -m
tricast_b200.serving`` prints that for every scheme. No TriCast counterpart (its cache emulation, ``src/tricast/kv/``,
has no attention of its own)."""

from __future__ import annotations

import torch

from .attention import paged_attention
from .kvcache import PagedKVCache
from .mma import gemm
from .norm import rms_norm_quantize
from .quantize import quantize
from .spec import get_preset


class AttentionLayer:
    """``w_qkv`` ``[(heads + 2 kv_heads) * head_dim, hidden]``, ``w_out`` ``[hidden, heads * head_dim]`` and the norm's
    ``gain`` ``[hidden]`` on the GPU. ``scheme``: of the GEMM operands (8-bit, with row or group scales);
    ``preset``: the accumulation rule of the GEMMs."""

    def __init__(self, w_qkv, w_out, gain, heads: int, kv_heads: int, *, scheme: str = "fp8_row",
                 preset: str = "nvidia_hopper_fp8", window: int = 0, eps: float = 1e-6):
        if heads < 1 or kv_heads < 1 or heads % kv_heads:
            raise ValueError("heads must be a multiple of kv_heads")
        if w_out.shape[1] % heads or w_qkv.shape != ((heads + 2 * kv_heads) * (w_out.shape[1] // heads), w_out.shape[0]):
            raise ValueError("w_qkv must have shape [(heads + 2 kv_heads) * head_dim, hidden], w_out [hidden, heads * head_dim]")
        self.heads, self.kv_heads, self.head_dim = heads, kv_heads, w_out.shape[1] // heads
        self.scheme, self.gain, self.window, self.eps, self.dtype = scheme, gain, window, eps, gain.dtype
        self.spec = get_preset(preset).with_(out_format="fp32")
        self.w_qkv, self.w_out = quantize(w_qkv, scheme), quantize(w_out, scheme)

    def __call__(self, x, residual, cache: PagedKVCache, slots, block_table, seq_lens, cu_q=None, *, max_q_len: int | None = None):
        """``(out, h)`` for the new tokens ``x`` ``[tokens, hidden]``: their keys and values go to ``slots`` of the
        cache, and they attend to the ``seq_lens`` tokens of their sequences (:func:`paged_attention`, which also says
        what ``cu_q`` and ``max_q_len`` are and default to). ``h`` is the residual stream, ``x + residual`` (``x`` itself
        without one)."""
        normed, h = rms_norm_quantize(x, self.gain, self.scheme, residual=residual, eps=self.eps)
        qkv = gemm(normed, self.w_qkv, self.spec).to(self.dtype).view(-1, self.heads + 2 * self.kv_heads, self.head_dim)
        q, k, v = qkv.split((self.heads, self.kv_heads, self.kv_heads), dim=1)  # views: strides are the operators' to follow
        cache.write(k, v, slots)
        a = paged_attention(q, cache, block_table, seq_lens, cu_q, max_q_len=max_q_len, window=self.window)
        out = gemm(quantize(a.view(a.shape[0], -1), self.scheme), self.w_out, self.spec).to(self.dtype)
        return out, x if residual is None else h


def run(cache_scheme, *, prompts=(200, 37), steps: int = 4, hidden: int = 512, heads: int = 8, kv_heads: int = 2,
        dtype=torch.bfloat16, page_size: int = 16, seed: int = 0) -> list:
    """Outputs of a layer on random data: one batch of prompts, then ``steps`` tokens for each of them."""
    g = torch.Generator(device="cuda").manual_seed(seed)

    def randn(*shape, scale=1.0):
        return (torch.randn(*shape, generator=g, device="cuda") * scale).to(dtype)

    dim, n = hidden // heads, len(prompts)
    layer = AttentionLayer(randn((heads + 2 * kv_heads) * dim, hidden, scale=hidden ** -0.5), randn(hidden, hidden, scale=hidden ** -0.5),
                           torch.ones(hidden, dtype=dtype, device="cuda"), heads, kv_heads)
    pages = -(-(max(prompts) + steps) // page_size)
    cache = PagedKVCache(n * pages, page_size, kv_heads, dim, cache_scheme, dtype=dtype)
    table = torch.randperm(n * pages, generator=g, device="cuda").to(torch.int32).view(n, pages)

    def slots(seq, first, count):
        at = torch.arange(first, first + count, device="cuda")
        return table[seq, at // page_size].long() * page_size + at % page_size

    lens = torch.tensor(prompts, dtype=torch.int32, device="cuda")
    cu = torch.nn.functional.pad(lens.cumsum(0), (1, 0)).to(torch.int32)
    where = torch.cat([slots(i, 0, p) for i, p in enumerate(prompts)])
    x, residual = randn(sum(prompts), hidden), randn(sum(prompts), hidden)
    outs = [layer(x, residual, cache, where, table, lens, cu, max_q_len=max(prompts))[0]]
    for t in range(steps):
        where = torch.cat([slots(i, p + t, 1) for i, p in enumerate(prompts)])
        x, residual = randn(n, hidden), randn(n, hidden)
        outs.append(layer(x, residual, cache, where, table, lens + t + 1)[0])
    return outs


def main() -> None:
    want = run(None)
    for scheme in ("fp8_row", "int8_row", "mxfp4"):
        got = run(scheme)
        db = [10 * torch.log10(w.double().square().sum() / (w.double() - o.double()).square().sum()).item() for w, o in zip(want, got)]
        print(f"{scheme:9s} SQNR against an unquantized cache: prompts {db[0]:.1f} dB, steps {min(db[1:]):.1f} dB at least")


if __name__ == "__main__":
    main()


__all__ = ["AttentionLayer", "run"]
