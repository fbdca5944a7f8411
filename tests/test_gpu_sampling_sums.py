"""What sampling adds up stays in 64 bits: weights that fp32 sums of a few neighbours would lose, in every place where sums are taken."""

from __future__ import annotations

import math

import numpy as np
import pytest
import torch

from tricast_b200 import sample_tokens

pytestmark = pytest.mark.gpu

# Weights 1 (logit 18.375), t (1) and t2 (0). 3 t is 8.5e-8, and both t and 2 t stay below half a step at 1, 6e-8: a sum of 1, t, t and t
# in fp32 is 1 in any order that begins with the 1.
TOP, T, T2 = 18.375, math.exp(-17.375), math.exp(-18.375)


def borders(count):
    """(quads of 1, t, t, t; quads of ones; u): of all weights the share s of the former is above u, but below it without the t's, by more than 4e-9
    each; weights good to 1.3e-7 move 3 t / 4 of a share by 3e-15."""
    found = []
    for a in range(2000, 2400):
        b = 800
        share, lost = (x / (x + 4 * b) for x in (a * (1 + 3 * T), a))
        u = np.float32((share + lost) / 2)
        if lost + 4e-9 < float(u) < share - 4e-9:
            found.append((a, b, float(u)))
    return found[:: len(found) // count][:count]


@pytest.mark.parametrize("vocab", [40000, 600000])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("last", ["all", "some", "unlike"])
def test_sums_of_what_is_kept(last, dtype, vocab):
    """top_k ends behind, or among, the four tokens of t2 that follow; those have one logit, or two whose weights are equal."""
    if last == "unlike" and dtype == torch.float16:
        pytest.skip("no two fp16 logits of this weight")
    cases = borders(6)
    assert len(cases) == 6
    z = torch.full((6, vocab), -math.inf)
    for row, (a, b, _) in zip(z, cases):
        row[:4 * a] = torch.tensor([TOP, 1.0, 1.0, 1.0]).repeat(a)
        row[4 * a:4 * (a + b)] = TOP
        row[4 * (a + b):4 * (a + b) + 4] = torch.tensor([0.0, 1e-10 if last == "unlike" else 0.0] * 2)
    z = z.to(dtype).cuda()
    u = torch.tensor([c[2] for c in cases], device="cuda")
    k = torch.tensor([4 * (a + b) + (4 if last == "all" else 2) for a, b, _ in cases], dtype=torch.int32, device="cuda")
    tokens, logprobs = sample_tokens(z, u, top_k=k, return_logprobs=True)
    assert tokens.tolist() == [4 * a - 4 for a, _, _ in cases]  # the last 1 that t's follow
    for got, (a, b, _) in zip(logprobs.tolist(), cases):
        want = -math.log(a * (1 + 3 * T) + 4 * b)
        assert abs(got - want) <= 2.0 ** -24 * abs(want) + 1e-9  # t2's four are 3e-12 of the sum


@pytest.mark.parametrize("vocab", [40000, 600000])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("with_k", [False, True])
def test_what_top_p_is_a_part_of(with_k, dtype, vocab):
    """A hair (2**-25) less than half of 8000 (1 + 3 t) is 4000.0001: 4001 tokens. Without the t's it is 3999.9998: 4000. With top_k the sum
    is of what that leaves, of t2's four tokens one."""
    a = 8000
    z = torch.full((1, vocab), -math.inf)
    z[0, :4 * a] = torch.tensor([TOP, 1.0, 1.0, 1.0]).repeat(a)
    z[0, 4 * a:4 * a + 4] = 0.0
    z = z.to(dtype).cuda()
    u = torch.tensor([1 - 2.0 ** -24], device="cuda")
    p = 0.5 - 2.0 ** -25
    assert p * a * (1 + 3 * T) > 4000 + 1e-4 and p * (a + 4 * T2) < 4000 - 2e-4
    token, logprob = sample_tokens(z, u, top_k=4 * a + 1 if with_k else None, top_p=p, return_logprobs=True)
    assert token.item() == 4 * 4000
    assert abs(logprob.item() + math.log(4001)) <= 2.0 ** -24 * math.log(4001) + 1e-9
