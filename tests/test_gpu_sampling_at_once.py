"""Sampling from several host threads: the library's calls run without Python's lock."""

from __future__ import annotations

import threading

import pytest
import torch

from tricast_b200 import _native, sample_tokens

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_threads_with_vocabularies_of_different_lengths(dtype):
    """A row of 150001 takes 75 KB of a block's shared memory, those of the other threads 4 and 16: what one launch asks for is not
    bounded by what another one needs. Through the C entry, whose calls then follow one another closely."""
    device, sizes, calls = torch.device("cuda", torch.cuda.current_device()), (150001, 1000, 150001, 4000), 10000
    sets = []
    for i, vocab in enumerate(sizes):
        g = torch.Generator(device="cuda").manual_seed(i)
        z = torch.randn(1, vocab, generator=g, device="cuda").to(dtype)
        u = torch.rand(1, generator=g, device="cuda")
        sets.append((z, u, sample_tokens(z, u, top_k=20), torch.empty(1, dtype=torch.int64, device="cuda")))
    torch.cuda.synchronize()
    lib, code = _native.lib(), _native.dtype_code(dtype)
    start, refused, wrong = threading.Barrier(len(sets)), [], []

    def work(z, u, want, out):
        with torch.cuda.device(device):
            stream = torch.cuda.Stream(device)
            args = (z.data_ptr(), code, 1, z.shape[1], z.shape[1], u.data_ptr(), None, 1.0, None, 20, None, 1.0, None, 0.0,
                    out.data_ptr(), None, stream.cuda_stream)
            start.wait(60)
            for _ in range(calls):
                if lib.tc_sample_tokens(*args):
                    refused.append(lib.tc_last_error())
            stream.synchronize()
            if not torch.equal(out, want):
                wrong.append((out.item(), want.item()))

    threads = [threading.Thread(target=work, args=s) for s in sets]
    for t in threads:
        t.start()
    for t in threads:
        t.join(120)
    assert not refused and not wrong, (len(refused), refused[:1], wrong)
