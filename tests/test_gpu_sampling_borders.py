"""Sampling where a token's place, 64 log2(e) (max - x) / temperature, rounds to the other side of a whole number.

The kernel counts tokens by such places in 32 bits and keeps what these lose
beside them. The logits here are searched for so that the place in 32 bits lies
across a whole number from the place itself, as far from it as its rounding
goes: what weighs is the place itself.

A weight is rounded to 2^-26 of what it is within 2^(1/64) of: off by at most
1.2 2^-27 of it, and so is a sum of weights. The logarithm of the largest one's
share, log(1 / sum), is off by as much, and by 2^-24 of itself from its rounding.
"""
import math

import pytest
import torch

from afterimage_amd.runtime.sampling import sample

pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.float16, torch.float32]
LATE = 1.0 - 2.0 ** -24  # draws the last token that is kept, of any that weighs 2^-23 of the sum


def across(dtype, up, low, high, seed):
    """(past, d, t): a logit's distance to the largest, a number of the type, and a temperature, for which the place lies by
    `past` below a whole number between low and high and its 32 bits at that or above (up), or the other way round; the worst
    of 60000."""
    g = torch.Generator().manual_seed(seed)
    d = (0.5 + 9.0 * torch.rand(60000, generator=g, dtype=torch.float64)).to(dtype).double()
    whole = torch.randint(low, high, (60000,), generator=g).double()
    aside = torch.exp2(-20.0 + 6.0 * torch.rand(60000, generator=g, dtype=torch.float64)) * (-1.0 if up else 1.0)
    t = 64.0 * math.log2(math.e) * d / (whole + aside)
    per = 64.0 * math.log2(math.e) / t
    place, rounded = d * per, (d.float() * per.float()).double()
    crosses = (place < whole) & (rounded >= whole) if up else (place >= whole) & (rounded < whole)
    past = torch.where(crosses, (whole - place).abs(), -1.0)
    i = int(past.argmax())
    assert float(past[i]) > 0, "none found"
    return float(past[i]), float(d[i]), float(t[i])


def row(dtype, d, equals, vocab):
    """The largest logit 0 at index 7, `equals` logits -d spread over the row, nothing else."""
    x = torch.full((vocab,), float("-inf"))
    at = torch.linspace(8, vocab - 1, equals).long()
    x[at] = -d
    x[7] = 0.0
    return x.to(dtype).cuda()[None], at


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("up", [True, False])
@pytest.mark.parametrize("equals,vocab,low,high", [(1000, 5000, 520, 700), (60000, 80000, 930, 1023), (100000, 120000, 1024, 1090), (260000, 262144, 1100, 1160)])
def test_sums_of_weights_whose_places_round_across(dtype, up, equals, vocab, low, high):
    """About half of the sum: the largest token's share says how far it is off."""
    _, d, t = across(dtype, up, low, high, vocab)
    x, _ = row(dtype, d, equals, vocab)
    token, log = sample(x, torch.zeros(1, device="cuda"), temperature=t, logprobs=True)
    want = -math.log1p(equals * math.exp(-d / t))
    assert int(token) == 7
    assert abs(float(log) - want) <= 1.2 * 2.0 ** -27 + 2.0 ** -24 * abs(want)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("up", [True, False])
@pytest.mark.parametrize("equals,vocab", [(1, 300), (40, 20000), (5000, 20000), (9, 100000), (5000, 100000)])
def test_min_p_between_a_place_and_its_rounding(dtype, up, equals, vocab):
    """min_p lies between what a token weighs and what its place in 32 bits would: the former decides. The place lies 2^-17 at
    least from the whole number, so a quarter of that from min_p's: 2^-19 ln 2 / 64, more than 2^-26, of the weight."""
    past, d, t = across(dtype, up, 700, 900, 3 * vocab + equals)
    assert past > 2.0 ** -17
    x, at = row(dtype, d, equals, vocab)
    place = d * 64.0 * math.log2(math.e) / t
    late = torch.full((1,), LATE, device="cuda")
    for move, kept in ((0.25, True), (0.75, True), (1.25, True), (-0.25, False), (-0.75, False), (-1.25, False)):
        least = 2.0 ** (-(place + move * past) / 64)
        got = int(sample(x, late, temperature=t, min_p=least))
        assert got == (int(at[-1]) if kept else 7), (move, got)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("up", [True, False])
def test_other_tokens_beside_those_across_a_border(dtype, up):
    """Tokens nearer and farther than the one across the border, top-k and top-p that end with it: order and sums go on."""
    _, d, t = across(dtype, up, 100, 250, 5)
    near = torch.tensor([0.0, 0.3 * d, 0.99 * d, d, d, 1.01 * d, 1.3 * d, 2.0 * d]).to(dtype)
    x = -near
    w = torch.exp(-near.double() / t)
    order = torch.sort(x.double(), descending=True, stable=True)[1]
    cum = w[order].cumsum(0)
    x = x.cuda()[None]
    for k in range(1, 9):
        for rank in range(k):
            # The middle of the token's part of the sum.
            u = torch.tensor([float((cum[rank] - w[order][rank] / 2) / cum[k - 1])], device="cuda")
            token, log = sample(x, u, temperature=t, top_k=k, logprobs=True)
            want = math.log(float(w[order][rank] / cum[k - 1]))
            assert int(token) == int(order[rank])
            assert abs(float(log) - want) <= 2.4 * 2.0 ** -27 + 2.0 ** -24 * abs(want)
        p = float((cum[k - 1] - w[order][k - 1] / 2) / cum[-1])
        assert int(sample(x, torch.full((1,), LATE, device="cuda"), temperature=t, top_p=p)) == int(order[k - 1])
