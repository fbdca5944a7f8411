"""CPU checks of the serving operators' C entries: the cache structure's layout, and arguments refused
before any device work."""

from __future__ import annotations

import ctypes
import subprocess
from pathlib import Path

import pytest

from tricast_b200 import _native as N
from tricast_b200.quantize import _qspec
from tricast_b200.spec import SCHEMES

ROOT = Path(__file__).resolve().parents[1]
P = ctypes.c_void_p(4096)  # never read: every call below is refused on the host


def test_cache_layout_matches_c(tmp_path):
    src = tmp_path / "sizes.c"
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "tricast_b200.h"\n'
                   'int main(void){printf("%zu %zu %zu\\n", sizeof(tc_kv_cache), offsetof(tc_kv_cache, num_pages), '
                   'offsetof(tc_kv_cache, head_dim));return 0;}\n')
    exe = tmp_path / "sizes"
    try:
        subprocess.run(["gcc", "-I", str(ROOT / "include"), str(src), "-o", str(exe)], check=True)
    except (OSError, subprocess.CalledProcessError):
        pytest.skip("no C compiler")
    want = list(map(int, subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.split()))
    assert [ctypes.sizeof(N.TcKvCache), N.TcKvCache.num_pages.offset, N.TcKvCache.head_dim.offset] == want


def _cache(**kw):
    c = N.TcKvCache()
    c.k = c.v = c.k_scale = c.v_scale = 4096
    c.scheme, c.dtype, c.num_pages, c.page_size, c.kv_heads, c.head_dim = 1, 1, 4, 16, 2, 64
    for name, value in kw.items():
        setattr(c, name, value)
    return c


@pytest.mark.parametrize("change", [dict(k=0), dict(v=0), dict(k_scale=0), dict(scheme=4), dict(dtype=3), dict(page_size=12),
                                    dict(page_size=512), dict(head_dim=24), dict(head_dim=272), dict(scheme=3, head_dim=48),
                                    dict(kv_heads=0), dict(num_pages=0), dict(k=4104)])
def test_cache_descriptors_are_checked(change):
    lib, c = N.lib(), _cache(**change)
    assert lib.tc_kv_write(c, P, 0, 0, P, 0, 0, P, 1, None) == N.TC_INVALID_ARGUMENT
    assert b"paged cache" in lib.tc_last_error()
    assert lib.tc_kv_read(c, P, 1, P, P, None) == N.TC_INVALID_ARGUMENT
    assert lib.tc_paged_attention(c, P, 64, 64, 1, 2, P, 1, 1, P, None, 1, 1, 1.0, 1, 0, P, None, None, 0,
                                  None) == N.TC_INVALID_ARGUMENT


def test_attention_arguments_are_checked():
    lib, c = N.lib(), _cache()

    def call(q=P, total=2, heads=4, table=P, pages=1, lens=P, cu=P, batch=1, max_q=2, scale=1.0, causal=1, window=0, out=P):
        return lib.tc_paged_attention(c, q, 256, 64, total, heads, table, 1, pages, lens, cu, batch, max_q, scale, causal,
                                      window, out, None, None, 0, None)

    for kw in (dict(q=None), dict(table=None), dict(lens=None), dict(out=None), dict(heads=3), dict(heads=0), dict(total=-1),
               dict(cu=None), dict(max_q=0), dict(scale=float("inf")), dict(window=-1), dict(window=4, causal=0),
               dict(pages=1 << 30), dict(batch=-1)):
        assert call(**kw) == N.TC_INVALID_ARGUMENT, kw
        assert lib.tc_last_error()


def test_norm_arguments_are_checked():
    lib = N.lib()

    def call(x=P, r=None, dtype=1, rows=2, K=64, xs=64, rs=64, w=P, wd=1, eps=1e-6, spec="fp8_row", codes=P, scale=P):
        return lib.tc_rms_norm_quantize(x, r, dtype, rows, K, xs, rs, w, wd, eps, _qspec(SCHEMES[spec]), codes, scale, None,
                                        None)

    for kw in (dict(x=None), dict(codes=None), dict(scale=None), dict(dtype=3), dict(wd=-1), dict(K=0), dict(xs=63),
               dict(r=P, rs=8), dict(eps=float("nan")), dict(eps=-1.0), dict(rows=-1), dict(rows=1 << 40)):
        assert call(**kw) == N.TC_INVALID_ARGUMENT, kw
    for spec in ("mxfp4", "nvfp4", "fp8_tensor", "fp8_block128", "bf16", "mxint8"):
        assert call(spec=spec) == N.TC_UNSUPPORTED, spec
    assert call(rows=0) == N.TC_OK
