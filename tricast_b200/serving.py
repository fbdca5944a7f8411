"""Layers as a server runs them: norm to an 8-bit operand, QKV GEMM, cache write, attention over the cache, output GEMM; norm,
gate and up GEMM, gated activation to an 8-bit operand, down GEMM; and a decoder of such layers that goes from the lengths of its
requests to their next tokens, with low-rank adapters for those that have one. The GEMMs follow an emulated accumulation rule
(attention's two products and the adapters' run on the tensor cores as they are). The module shows the serving operators together
and measures what a cache scheme costs end to end; ``python -m tricast_b200.serving`` prints that for every scheme. No TriCast
counterpart (its cache emulation, ``src/tricast/kv/``, has no attention of its own)."""

from __future__ import annotations

from typing import NamedTuple

import torch

from .adapters import low_rank_add
from .attention import paged_attention
from .gated import gated_quantize
from .kvcache import PagedKVCache
from .mma import gemm
from .norm import rms_norm_quantize
from .paging import plan_pages, release_pages
from .quantize import quantize
from .sampling import sample_tokens
from .spec import get_preset


class Adapters(NamedTuple):
    """Low-rank adapters of one projection, as :func:`low_rank_add` takes them."""

    a: torch.Tensor  # [adapters, rank, k]
    b: torch.Tensor  # [adapters, n, rank]
    gain: torch.Tensor | None = None  # fp32 [adapters]


def _project(x, operand, weight, spec, dtype, adapters, index):
    """``operand`` times ``weight`` in ``dtype``, with the adapters' products of ``x`` on top where there are some."""
    y = gemm(operand, weight, spec)
    if adapters is None or index is None:  # rounded as with an index: what a token without an adapter gets does not depend on it
        return y.to(dtype)
    return low_rank_add(y, x, adapters.a, adapters.b, index, gain=adapters.gain, dtype=dtype)


class AttentionLayer:
    """``w_qkv`` ``[(heads + 2 kv_heads) * head_dim, hidden]``, ``w_out`` ``[hidden, heads * head_dim]`` and the norm's
    ``gain`` ``[hidden]`` on the GPU. ``scheme``: of the GEMM operands (8-bit, with row or group scales);
    ``preset``: the accumulation rule of the GEMMs. ``qkv_adapters``, ``out_adapters``: low-rank adapters beside the two
    projections (the first reads the norm's operand, whose scales are then per row)."""

    def __init__(self, w_qkv, w_out, gain, heads: int, kv_heads: int, *, scheme: str = "fp8_row",
                 preset: str = "nvidia_hopper_fp8", window: int = 0, eps: float = 1e-6,
                 qkv_adapters: Adapters | None = None, out_adapters: Adapters | None = None):
        if heads < 1 or kv_heads < 1 or heads % kv_heads:
            raise ValueError("heads must be a multiple of kv_heads")
        if w_out.shape[1] % heads or w_qkv.shape != ((heads + 2 * kv_heads) * (w_out.shape[1] // heads), w_out.shape[0]):
            raise ValueError("w_qkv must have shape [(heads + 2 kv_heads) * head_dim, hidden], w_out [hidden, heads * head_dim]")
        self.heads, self.kv_heads, self.head_dim = heads, kv_heads, w_out.shape[1] // heads
        self.scheme, self.gain, self.window, self.eps, self.dtype = scheme, gain, window, eps, gain.dtype
        self.spec = get_preset(preset).with_(out_format="fp32")
        self.w_qkv, self.w_out = quantize(w_qkv, scheme), quantize(w_out, scheme)
        self.qkv_adapters, self.out_adapters = qkv_adapters, out_adapters

    def __call__(self, x, residual, cache: PagedKVCache, slots, block_table, seq_lens, cu_q=None, *, max_q_len: int | None = None,
                 index=None):
        """``(out, h)`` for the new tokens ``x`` ``[tokens, hidden]``: their keys and values go to ``slots`` of the
        cache, and they attend to the ``seq_lens`` tokens of their sequences (:func:`paged_attention`, which also says
        what ``cu_q`` and ``max_q_len`` are and default to). ``index`` (int32 ``[tokens]``): each token's adapter, ``-1``
        for none. ``h`` is the residual stream, ``x + residual`` (``x`` itself without one)."""
        normed, h = rms_norm_quantize(x, self.gain, self.scheme, residual=residual, eps=self.eps)
        qkv = _project(normed, normed, self.w_qkv, self.spec, self.dtype, self.qkv_adapters, index)
        qkv = qkv.view(-1, self.heads + 2 * self.kv_heads, self.head_dim)
        q, k, v = qkv.split((self.heads, self.kv_heads, self.kv_heads), dim=1)  # views: strides are the operators' to follow
        cache.write(k, v, slots)
        a = paged_attention(q, cache, block_table, seq_lens, cu_q, max_q_len=max_q_len, window=self.window)
        a = a.view(a.shape[0], -1)
        out = _project(a, quantize(a, self.scheme), self.w_out, self.spec, self.dtype, self.out_adapters, index)
        return out, x if residual is None else h


class FeedForwardLayer:
    """``w_gate_up`` ``[2 * inner, hidden]`` (the gate's rows first), ``w_down`` ``[hidden, inner]`` and the norm's ``gain``
    ``[hidden]`` on the GPU; ``activation`` as :func:`gated_quantize` names it, the rest as for :class:`AttentionLayer`. Both adapters read
    8-bit operands, whose scales are then per row. A layer with ``gate_up_adapters`` rounds gate and up to ``gain``'s dtype before the
    activation, for tokens without an adapter and calls without ``index`` too; one without them keeps the GEMM's fp32."""

    def __init__(self, w_gate_up, w_down, gain, *, activation: str = "silu", scheme: str = "fp8_row",
                 preset: str = "nvidia_hopper_fp8", eps: float = 1e-6, gate_up_adapters: Adapters | None = None,
                 down_adapters: Adapters | None = None):
        self.inner = w_down.shape[1]
        if w_gate_up.shape != (2 * self.inner, w_down.shape[0]):
            raise ValueError("w_gate_up must have shape [2 * inner, hidden], w_down [hidden, inner]")
        self.scheme, self.gain, self.eps, self.activation, self.dtype = scheme, gain, eps, activation, gain.dtype
        self.spec = get_preset(preset).with_(out_format="fp32")
        self.w_gate_up, self.w_down = quantize(w_gate_up, scheme), quantize(w_down, scheme)
        self.gate_up_adapters, self.down_adapters = gate_up_adapters, down_adapters

    def __call__(self, x, residual, *, index=None):
        """``(out, h)`` for the tokens ``x`` ``[tokens, hidden]``, ``index`` and ``h`` as for :class:`AttentionLayer`."""
        normed, h = rms_norm_quantize(x, self.gain, self.scheme, residual=residual, eps=self.eps)
        wide = torch.float32 if self.gate_up_adapters is None else self.dtype
        y = _project(normed, normed, self.w_gate_up, self.spec, wide, self.gate_up_adapters, index)
        gated = gated_quantize(y[:, :self.inner], y[:, self.inner:], self.scheme, activation=self.activation)
        out = _project(gated, gated, self.w_down, self.spec, self.dtype, self.down_adapters, index)
        return out, x if residual is None else h


class Decoder:
    """``layers`` (pairs of an :class:`AttentionLayer` and a :class:`FeedForwardLayer`) between an ``embedding`` ``[vocab, hidden]``
    and a ``head`` ``[vocab, hidden]`` behind a last norm's ``gain`` ``[hidden]``."""

    def __init__(self, embedding, layers, gain, head, *, scheme: str = "fp8_row", preset: str = "nvidia_hopper_fp8", eps: float = 1e-6):
        if head.shape[1:] != embedding.shape[1:] or head.shape[0] > embedding.shape[0]:  # a drawn token is looked up next
            raise ValueError("head must be [vocab, hidden] with no more rows than the embedding")
        self.embedding, self.layers, self.gain, self.scheme, self.eps = embedding, layers, gain, scheme, eps
        self.spec = get_preset(preset).with_(out_format="fp32")
        self.head = quantize(head, scheme)

    def __call__(self, tokens, caches, plan, block_table, *, max_q_len: int | None = None, index=None):
        """fp32 logits ``[batch, vocab]`` behind the last of each sequence's new ``tokens`` (int64 ``[tokens]``, as many as the plan has
        room for, in its order; what stands behind the plan's last one does not matter, the others must lie in the vocabulary).
        ``plan``: of :func:`plan_pages` for them. A sequence without new tokens has some other's logits."""
        if len(caches) != len(self.layers):
            raise ValueError("a decoder needs a cache for each of its layers")
        if tokens.shape != plan.sequence.shape:
            raise ValueError("tokens must be as many as the plan has room for")
        x, h = self.embedding[torch.where(plan.sequence < 0, 0, tokens)], None
        for cache, (attention, feed_forward) in zip(caches, self.layers):
            x, h = attention(x, h, cache, plan.slots, block_table, plan.seq_lens, plan.cu_q, max_q_len=max_q_len, index=index)
            x, h = feed_forward(x, h, index=index)
        last = (plan.cu_q[1:].long() - 1).clamp(min=0)
        normed, _ = rms_norm_quantize(x[last], self.gain, self.scheme, residual=h[last], eps=self.eps)
        return gemm(normed, self.head, self.spec)


def generate(decoder: Decoder, prompts, steps: int, cache_scheme=None, *, uniform=None, page_size: int = 16, adapter=None,
             temperature=1.0, top_k=None, top_p=None, min_p=None):
    """int64 ``[batch, steps]``: what the decoder says after each of ``prompts`` (lists of token ids). ``uniform``: the random numbers, fp32
    ``[steps, batch]`` (torch's default generator without them); ``adapter``: int32 ``[batch]``, each request's adapter;
    the rest as :func:`sample_tokens` takes it. A request whose logits have no token (:func:`sample_tokens` says -1) gets no more
    of them: -1 from there on. Page tables, slots, positions and tokens stay on the GPU."""
    device = decoder.gain.device
    batch, lens = len(prompts), [len(p) for p in prompts]
    if batch == 0 or min(lens) == 0 or steps < 1:
        raise ValueError("generate needs prompts of one token at least, and steps")
    vocab = decoder.embedding.shape[0]
    if any(not 0 <= t < vocab for p in prompts for t in p):
        raise ValueError(f"prompts hold token ids from 0 to {vocab - 1}")
    if adapter is not None and (adapter.shape != (batch,) or adapter.dtype != torch.int32 or adapter.device != device):
        raise ValueError("adapter must be an int32 tensor [batch] on the decoder's device")
    if uniform is not None and (uniform.ndim != 2 or uniform.shape[0] < steps or uniform.shape[1] != batch):
        raise ValueError("uniform must be a tensor [steps, batch]")
    width = -(-(max(lens) + steps) // page_size)
    pages = sum(-(-(n + steps) // page_size) for n in lens)
    caches = [PagedKVCache(pages, page_size, attention.kv_heads, attention.head_dim, cache_scheme, dtype=attention.dtype, device=device)
              for attention, _ in decoder.layers]
    as32 = dict(dtype=torch.int32, device=device)
    table, free, taken = torch.full((batch, width), -1, **as32), torch.arange(pages, **as32), torch.zeros(1, **as32)
    new, have = torch.tensor(lens, **as32), torch.zeros(batch, **as32)
    tokens = torch.tensor([t for p in prompts for t in p], dtype=torch.int64, device=device)
    if uniform is None:
        uniform = torch.rand(steps, batch, device=device)
    said = torch.empty(steps, batch, dtype=torch.int64, device=device)
    for step in range(steps):
        plan = plan_pages(have, new, table, free, taken, page_size=page_size, tokens=tokens.shape[0] if step == 0 else batch)
        owner = plan.sequence.clamp(min=0).long()
        if step:
            tokens = said[step - 1][owner]  # those that go on stand side by side
        index = None if adapter is None else adapter[owner]
        logits = decoder(tokens, caches, plan, table, max_q_len=max(lens) if step == 0 else 1, index=index)
        got = sample_tokens(logits, uniform[step], temperature=temperature, top_k=top_k, top_p=top_p, min_p=min_p)
        said[step] = torch.where(new > 0, got, -1)
        have, taken, new = plan.seq_lens, plan.taken, (said[step] >= 0).to(torch.int32)
    release_pages(table, torch.ones(batch, dtype=torch.bool, device=device), free, taken)
    return said.t()


def random_decoder(*, vocab: int = 1024, hidden: int = 256, heads: int = 4, kv_heads: int = 2, inner: int = 512, layers: int = 2,
                   dtype=torch.bfloat16, seed: int = 0, adapters: int = 0, rank: int = 8, scheme: str = "fp8_row") -> Decoder:
    """A decoder with random weights, and with ``adapters`` random adapters beside every projection."""
    g = torch.Generator(device="cuda").manual_seed(seed)

    def randn(*shape, scale=1.0):
        return (torch.randn(*shape, generator=g, device="cuda") * scale).to(dtype)

    def beside(k, n):
        return Adapters(randn(adapters, rank, k, scale=k ** -0.5), randn(adapters, n, rank, scale=0.2)) if adapters else None

    dim, ones = hidden // heads, torch.ones(hidden, dtype=dtype, device="cuda")
    qkv = (heads + 2 * kv_heads) * dim
    pairs = [(AttentionLayer(randn(qkv, hidden, scale=hidden ** -0.5), randn(hidden, heads * dim, scale=hidden ** -0.5), ones, heads, kv_heads,
                             scheme=scheme, qkv_adapters=beside(hidden, qkv), out_adapters=beside(heads * dim, hidden)),
              FeedForwardLayer(randn(2 * inner, hidden, scale=hidden ** -0.5), randn(hidden, inner, scale=inner ** -0.5), ones, scheme=scheme,
                               gate_up_adapters=beside(hidden, 2 * inner), down_adapters=beside(inner, hidden)))
             for _ in range(layers)]
    return Decoder(randn(vocab, hidden), pairs, ones, randn(vocab, hidden, scale=hidden ** -0.5), scheme=scheme)


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
    as32 = dict(dtype=torch.int32, device="cuda")
    free = torch.randperm(n * pages, generator=g, device="cuda").to(torch.int32)
    table, lens = torch.full((n, pages), -1, **as32), torch.tensor(prompts, **as32)
    plan = plan_pages(torch.zeros(n, **as32), lens, table, free, torch.zeros(1, **as32), page_size=page_size, tokens=sum(prompts))
    x, residual = randn(sum(prompts), hidden), randn(sum(prompts), hidden)
    outs = [layer(x, residual, cache, plan.slots, table, plan.seq_lens, plan.cu_q, max_q_len=max(prompts))[0]]
    one = torch.ones(n, **as32)
    for _ in range(steps):
        plan = plan_pages(plan.seq_lens, one, table, free, plan.taken, page_size=page_size, tokens=n)
        x, residual = randn(n, hidden), randn(n, hidden)
        outs.append(layer(x, residual, cache, plan.slots, table, plan.seq_lens)[0])
    return outs


def main() -> None:
    want = run(None)
    for scheme in ("fp8_row", "int8_row", "mxfp4"):
        got = run(scheme)
        db = [10 * torch.log10(w.double().square().sum() / (w.double() - o.double()).square().sum()).item() for w, o in zip(want, got)]
        print(f"{scheme:9s} SQNR against an unquantized cache: prompts {db[0]:.1f} dB, steps {min(db[1:]):.1f} dB at least")
    decoder = random_decoder(adapters=3)
    prompts = [list(range(i, 40 * (i + 1))) for i in range(16)]
    settings = dict(uniform=torch.rand(24, 16, generator=torch.Generator().manual_seed(1)).cuda(), temperature=0.7, top_k=50, top_p=0.95,
                    adapter=torch.arange(16, dtype=torch.int32, device="cuda") % 4 - 1)
    want = generate(decoder, prompts, 24, **settings)
    for scheme in ("fp8_row", "int8_row", "mxfp4"):
        same = (generate(decoder, prompts, 24, scheme, **settings) == want).to(torch.int32).cumprod(1).sum(1)
        print(f"{scheme:9s} tokens that equal those of an unquantized cache before the first that differs: {same.double().mean():.1f} of 24")


if __name__ == "__main__":
    main()


__all__ = ["Adapters", "AttentionLayer", "Decoder", "FeedForwardLayer", "generate", "random_decoder", "run"]
