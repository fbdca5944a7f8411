"""Requests that generate refuses, and those whose logits have no token."""

from __future__ import annotations

import pytest
import torch

from tricast_b200 import serving
from tricast_b200.serving import Decoder, generate, random_decoder


def unbuilt():
    d = Decoder.__new__(Decoder)
    d.gain, d.embedding, d.layers = torch.ones(4), torch.ones(10, 4), []
    return d


@pytest.mark.parametrize("prompts", [[[1, 10]], [[0], [-1]], [[2 ** 40]]])
def test_ids_outside_the_vocabulary_are_refused(prompts):
    with pytest.raises(ValueError, match="token ids"):
        generate(unbuilt(), prompts, 1)


def test_settings_of_another_batch_are_refused():
    prompts = [[1], [2, 3]]
    for adapter in (torch.zeros(1, dtype=torch.int32), torch.zeros(3, dtype=torch.int32), torch.zeros(2, dtype=torch.int64),
                    torch.zeros(2, 1, dtype=torch.int32)):
        with pytest.raises(ValueError, match="adapter"):
            generate(unbuilt(), prompts, 1, adapter=adapter)
    for uniform in (torch.zeros(2), torch.zeros(1, 2), torch.zeros(3, 1)):
        with pytest.raises(ValueError, match="uniform"):
            generate(unbuilt(), prompts, 2, uniform=uniform)


@pytest.mark.gpu
@pytest.mark.parametrize("adapters", [0, 2])
def test_a_request_without_a_token_ends_alone(monkeypatch, adapters):
    """Sampling says -1 for requests 1 and 3 after some steps, whatever it says later: they stay at -1, and the others say what they say
    with them (in fp32, where every row of every operator is computed by itself)."""
    decoder = random_decoder(vocab=300, hidden=64, heads=2, kv_heads=1, inner=96, dtype=torch.float32, adapters=adapters, seed=3)
    prompts, steps = [[5, 9, 2], [7] * 18, [1], [4, 4]], 7
    uniform = torch.rand(steps, 4, generator=torch.Generator().manual_seed(2)).cuda()
    settings = dict(uniform=uniform, page_size=8, temperature=0.8, top_p=0.9)
    if adapters:
        settings["adapter"] = torch.tensor([1, -1, 0, 1], dtype=torch.int32, device="cuda")
    want = generate(decoder, prompts, steps, None, **settings)
    real, calls = serving.sample_tokens, []

    def sample(*args, **kw):
        got = real(*args, **kw)
        calls.append(len(calls))
        got[1] = -1 if len(calls) == 1 else got[1]
        got[3] = -1 if len(calls) == 4 else got[3]
        return got

    monkeypatch.setattr(serving, "sample_tokens", sample)
    got = generate(decoder, prompts, steps, None, **settings)
    assert torch.equal(got[[0, 2]], want[[0, 2]])
    assert (got[1] == -1).all()
    assert torch.equal(got[3, :3], want[3, :3]) and (got[3, 3:] == -1).all()


@pytest.mark.gpu
def test_requests_that_are_not_numbers():
    """An embedding of NaN gives its request no token, and the others theirs."""
    decoder = random_decoder(vocab=300, hidden=64, heads=2, kv_heads=1, inner=96, dtype=torch.float32, seed=3)
    uniform = torch.rand(4, 3, generator=torch.Generator().manual_seed(2)).cuda()
    want = generate(decoder, [[5, 9], [8, 1], [6]], 4, None, uniform=uniform, top_k=30)
    decoder.embedding[299] = float("nan")
    got = generate(decoder, [[5, 9], [8, 299], [6]], 4, None, uniform=uniform, top_k=30)
    assert not (want[[0, 2]] == 299).any()  # or they would have met it too
    assert torch.equal(got[[0, 2]], want[[0, 2]]) and (got[1] == -1).all()
