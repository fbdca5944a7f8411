"""CPU checks of the C entries of page plans, adapters, the gated activation and sampling: arguments refused before any
device work, and what Python refuses without a GPU."""

from __future__ import annotations

import ctypes

import pytest
import torch

from tricast_b200 import _native as N
from tricast_b200 import gated_quantize, low_rank_add, plan_pages, release_pages, sample_tokens
from tricast_b200.quantize import _qspec
from tricast_b200.spec import SCHEMES

P = ctypes.c_void_p(4096)  # never read: every call below is refused on the host
BAD = N.TC_INVALID_ARGUMENT


def test_plan_arguments_are_checked():
    lib = N.lib()
    assert lib.tc_plan_pages_workspace(-1) == 0 and lib.tc_plan_pages_workspace(3000) >= 24000

    def call(lens=P, new=P, batch=3, table=P, stride=4, width=4, free=P, nfree=8, taken=P, page=16, tokens=5, out=P, cu=P,
             slots=P, seq=P, pos=P, top=P, missing=P, ws=P, nbytes=1 << 12):
        return lib.tc_plan_pages(lens, new, batch, table, stride, width, free, nfree, taken, page, tokens, out, cu, slots, seq,
                                 pos, top, missing, ws, nbytes, None)

    for kw in (dict(lens=None), dict(new=None), dict(table=None), dict(free=None), dict(taken=None), dict(out=None),
               dict(cu=None), dict(slots=None), dict(seq=None), dict(pos=None), dict(top=None), dict(missing=None),
               dict(batch=-1), dict(width=-1), dict(tokens=-1), dict(nfree=-1), dict(page=0), dict(page=12), dict(stride=3),
               dict(tokens=1 << 31), dict(nfree=1 << 31), dict(width=1 << 27, stride=1 << 27)):
        assert call(**kw) == BAD, kw
        assert b"tc_plan_pages" in lib.tc_last_error()
    assert call(batch=3000, ws=None) == N.TC_WORKSPACE_TOO_SMALL and call(batch=3000, nbytes=8) == N.TC_WORKSPACE_TOO_SMALL


def test_release_arguments_are_checked():
    lib = N.lib()

    def call(table=P, stride=4, width=4, ended=P, batch=3, free=P, nfree=8, taken=P, top=P, ws=P, nbytes=1 << 12):
        return lib.tc_release_pages(table, stride, width, ended, batch, free, nfree, taken, top, ws, nbytes, None)

    for kw in (dict(table=None), dict(ended=None), dict(free=None), dict(taken=None), dict(top=None), dict(stride=3),
               dict(batch=-1), dict(width=-1), dict(nfree=-1), dict(nfree=1 << 31)):
        assert call(**kw) == BAD, kw
        assert b"tc_release_pages" in lib.tc_last_error()
    assert call(ws=None) == N.TC_WORKSPACE_TOO_SMALL and call(nbytes=4) == N.TC_WORKSPACE_TOO_SMALL


def test_adapter_arguments_are_checked():
    lib = N.lib()

    def call(y=P, yd=0, ys=64, x=P, xk=1, xs=32, scale=None, tokens=2, k=32, n=64, a=P, b=P, wd=1, adapters=3, rank=8, gain=None,
             index=P, out=P, od=1):
        return lib.tc_low_rank_add(y, yd, ys, x, xk, xs, scale, tokens, k, n, a, b, wd, adapters, rank, gain, index, out, od, None, 0, None)

    for kw in (dict(y=None), dict(x=None), dict(a=None), dict(b=None), dict(index=None), dict(out=None), dict(yd=3), dict(xk=6),
               dict(xk=-1), dict(wd=3), dict(od=-1), dict(ys=63), dict(xs=31), dict(xk=3), dict(tokens=-1), dict(k=-1),
               dict(n=-1), dict(rank=0), dict(rank=1025), dict(adapters=-1), dict(tokens=1 << 31), dict(n=1 << 31, ys=1 << 31)):
        assert call(**kw) == BAD, kw
        assert b"tc_low_rank_add" in lib.tc_last_error()
    assert call(tokens=0) == N.TC_OK and call(n=0) == N.TC_OK


def test_gated_arguments_are_checked():
    lib = N.lib()

    def call(g=P, gs=64, u=P, us=64, dtype=1, rows=2, K=64, act=0, spec="fp8_row", codes=P, scale=P):
        return lib.tc_gated_quantize(g, gs, u, us, dtype, rows, K, act, _qspec(SCHEMES[spec]), codes, scale, None)

    for kw in (dict(g=None), dict(u=None), dict(codes=None), dict(scale=None), dict(dtype=3), dict(act=4), dict(act=-1),
               dict(K=0), dict(gs=63), dict(us=63), dict(rows=-1), dict(rows=1 << 40)):
        assert call(**kw) == BAD, kw
        assert b"tc_gated_quantize" in lib.tc_last_error()
    for spec in ("mxfp4", "nvfp4", "fp8_tensor", "fp8_block128", "bf16", "mxint8"):
        assert call(spec=spec) == N.TC_UNSUPPORTED, spec
    assert call(rows=0) == N.TC_OK


def test_sampling_arguments_are_checked():
    lib = N.lib()

    def call(z=P, dtype=0, rows=2, vocab=8, stride=8, u=P, tokens=P):
        return lib.tc_sample_tokens(z, dtype, rows, vocab, stride, u, None, 1.0, None, 0, None, 1.0, None, 0.0, tokens, None, None)

    for kw in (dict(z=None), dict(u=None), dict(tokens=None), dict(dtype=3), dict(rows=-1), dict(rows=1 << 28), dict(vocab=0),
               dict(vocab=1 << 31), dict(stride=7)):
        assert call(**kw) == BAD, kw
        assert b"tc_sample_tokens" in lib.tc_last_error()
    assert call(rows=0) == N.TC_OK


def test_tensors_of_the_host_are_refused():
    i = torch.zeros(2, dtype=torch.int32)
    table = torch.zeros(2, 4, dtype=torch.int32)
    x = torch.zeros(2, 64)
    for call in (lambda: plan_pages(i, i, table, i, i[:1], page_size=16, tokens=2),
                 lambda: release_pages(table, i.bool(), i, i[:1]),
                 lambda: low_rank_add(x, x, x.view(1, 2, 64), x.view(1, 64, 2), i),
                 lambda: gated_quantize(x, x, "fp8_row"),
                 lambda: sample_tokens(x, x[:, 0])):
        with pytest.raises(ValueError, match="CUDA"):
            call()
    with pytest.raises(ValueError, match="activation"):
        gated_quantize(x, x, "fp8_row", activation="tanh")
    with pytest.raises(NotImplementedError):
        gated_quantize(x, x, "bf16")
