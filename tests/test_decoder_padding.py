"""Token ids behind a plan's last token, without a GPU: they are never looked up."""

from __future__ import annotations

import pytest
import torch

from tricast_b200.paging import PagePlan
from tricast_b200.serving import Decoder


class Reached(Exception):
    pass


def decoder(vocab=10, layers=1):
    def attention(x, *args, **kw):
        raise Reached(x)

    d = Decoder.__new__(Decoder)
    d.embedding, d.layers = torch.arange(float(vocab))[:, None].expand(vocab, 4), [(attention, None)] * layers
    return d


def plan(sequence):
    return PagePlan(None, None, None, torch.tensor(sequence, dtype=torch.int32), None, None, None)


@pytest.mark.parametrize("padding", [0, 9, -1, 10, -11, 2 ** 40, -2 ** 63])
def test_padding_may_hold_anything(padding):
    tokens = torch.tensor([3, 9, 0, padding, padding])
    with pytest.raises(Reached) as e:
        decoder()(tokens, [None], plan([0, 0, 2, -1, -1]), None)
    x = e.value.args[0]
    assert x.shape == (5, 4) and x[:3, 0].tolist() == [3.0, 9.0, 0.0]


def test_sizes_that_do_not_fit():
    with pytest.raises(ValueError, match="plan has room"):
        decoder()(torch.tensor([1, 2, 3]), [None], plan([0, 0]), None)
    with pytest.raises(ValueError, match="cache"):
        decoder(layers=2)(torch.tensor([1, 2]), [None], plan([0, 0]), None)


def test_a_head_of_another_vocabulary_is_refused():
    for head in (torch.ones(12, 4), torch.ones(10, 8), torch.ones(10)):
        with pytest.raises(ValueError, match="no more rows"):
            Decoder(torch.ones(10, 4), [], torch.ones(4), head)
