"""Tokens from logits against the definition in 64 bits.

A weight is rounded to 2^-26 of its bin's top, which it is within 2^(1/64) of,
and its series is off by less than 2^-30: at most 1.2 2^-27 of it, and so is any
sum of weights of itself. Where a prefix ends and where the draw falls are
comparisons of two such sums, so borders move by less than 2^-25 of the whole: a
row's token has to lie between those of borders moved that far either way (the
same one, for most rows). The logarithm of a share is off by 2^-25 from its
weights, by its sum's own ends, and 2^-24 of itself from its rounding.
"""
import math

import pytest
import torch

from afterimage_amd.runtime.sampling import sample

pytestmark = pytest.mark.gpu

NEAR = 2.0 ** -25


def define(x, u, t, k, p, m):
    """One row in 64 bits, on the CPU: its tokens in order, the first and last rank that may be drawn, every rank's weight, and
    the least and most that the kept ones may weigh in all."""
    x = torch.where(x.isnan(), float("-inf"), x.double().cpu())
    order = torch.sort(x, descending=True, stable=True)[1]
    x = x[order]
    if x[0] == float("-inf"):
        return None
    if not t > 0:
        k, t = 1, 1.0
    w = torch.where(x == x[0], 1.0, torch.exp((x - x[0]) / t))
    if k > 0:
        w[k:] = 0
    cum = w.cumsum(0)
    heavy = int((w >= min(m, 1.0)).sum()) if m > 0 else int((w > 0).sum())
    ends = []
    for move in (-NEAR, NEAR):
        n = int((cum - w < (max(p, 0.0) + move) * float(cum[-1])).sum()) if p < 1 else len(w)
        ends.append(max(1, min(n, heavy)))
    low, high = (float(cum[n - 1]) for n in ends)
    first = int((cum <= u * low - NEAR * high).sum())
    last = min(int((cum <= u * high + NEAR * high).sum()), ends[1] - 1)
    return order, min(first, ends[0] - 1), last, w, low, high


def compare(logits, u, t=1.0, k=0, p=1.0, m=0.0):
    tokens, logs = sample(logits, u, temperature=t, top_k=k, top_p=p, min_p=m, logprobs=True)
    assert torch.equal(tokens, sample(logits, u, temperature=t, top_k=k, top_p=p, min_p=m))
    n = logits.shape[0]
    each = [x.tolist() if isinstance(x, torch.Tensor) else [x] * n for x in (u, t, k, p, m)]
    rows = logits.cpu()
    for r, setting in enumerate(zip(*each)):
        found = define(rows[r], *setting)
        got, log = int(tokens[r]), float(logs[r])
        if found is None:
            assert got == -1 and log == float("-inf"), "row %d" % r
            continue
        order, first, last, w, low, high = found
        ranks = [i for i in range(first, last + 1) if int(order[i]) == got]
        assert ranks, "row %d: %d is not among %s" % (r, got, order[first:last + 1].tolist()[:5])
        least, most = math.log(float(w[ranks[0]]) / high), math.log(float(w[ranks[0]]) / low)
        room = 2.0 ** -25 + 2.0 ** -24 * abs(least)
        assert least - room <= log <= most + room, "row %d" % r
    return tokens


def inputs(rows, vocab, dtype, spread=2.5, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(rows, vocab, generator=g, device="cuda") * spread
    return x.to(dtype), torch.rand(rows, generator=g, device="cuda")


DTYPES = [torch.bfloat16, torch.float16, torch.float32]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("vocab", [1, 2, 7, 63, 500, 4097, 32000, 50001])
def test_every_rule_and_none(dtype, vocab):
    x, u = inputs(6, vocab, dtype, seed=vocab)
    for t, k, p, m in [(1.0, 0, 1.0, 0.0), (0.7, 0, 0.9, 0.0), (1.3, 20, 1.0, 0.0), (0.5, 0, 1.0, 0.05), (0.9, 40, 0.8, 0.02), (0.0, 5, 0.5, 0.1),
                       (1.0, 1, 1.0, 0.0), (1.0, 0, 0.0, 0.0), (1.0, 0, 1.0, 1.0), (1.0, 10 ** 9, 0.999, 1e-6)]:
        compare(x, u, t, k, p, m)


@pytest.mark.parametrize("dtype", DTYPES)
def test_large_vocabularies(dtype):
    for vocab, rows in ((151936, 8), (262144, 3)):
        x, u = inputs(rows, vocab, dtype, seed=rows)
        for t, k, p, m in [(1.0, 0, 1.0, 0.0), (0.8, 50, 0.95, 0.0), (1.0, 0, 0.9, 0.0), (0.6, 0, 1.0, 0.02), (1.5, 2000, 0.99, 0.0)]:
            compare(x, u, t, k, p, m)


@pytest.mark.parametrize("rows", [64, 65])
def test_many_rows_of_a_large_vocabulary(rows):
    """On both sides of where a row's work is dealt out."""
    x, u = inputs(rows, 90001, torch.bfloat16, seed=rows)
    for t, k, p, m in [(1.0, 0, 0.9, 0.0), (0.8, 50, 0.95, 0.01)]:
        compare(x, u, t, k, p, m)


def test_settings_of_their_own_for_each_row():
    x, u = inputs(40, 3001, torch.float32, seed=4)
    g = torch.Generator().manual_seed(4)
    t = torch.tensor([0.0, 0.3, 0.7, 1.0, 2.0])[torch.randint(5, (40,), generator=g)].cuda()
    k = torch.tensor([-3, 0, 1, 7, 5000], dtype=torch.int32)[torch.randint(5, (40,), generator=g)].cuda()
    p = torch.tensor([0.25, 0.9, 1.0, 3.0])[torch.randint(4, (40,), generator=g)].cuda()
    m = torch.tensor([-1.0, 0.0, 0.01, 0.5])[torch.randint(4, (40,), generator=g)].cuda()
    compare(x, u, t, k, p, m)


def test_numbers_out_of_range():
    """Mean the nearest in it: NaN and negative temperatures the largest logit, NaN elsewhere no rule or the first token."""
    x, _ = inputs(6, 300, torch.float32, seed=6)
    nan, inf = float("nan"), float("inf")
    top = x.argmax(1)
    u = torch.tensor([0.5] * 6, device="cuda")
    assert torch.equal(sample(x, u, temperature=torch.tensor([nan, -1.0, 0.0, -inf, 0.0, nan], device="cuda")), top)
    assert torch.equal(sample(x, torch.tensor([-1.0, nan, 0.0, -inf, 0.0, -0.0], device="cuda")), top)
    last = sample(x, torch.tensor([1.0, 2.0, inf, 1.0, 1.0, 1.0], device="cuda"), top_k=5)
    assert torch.equal(last, torch.sort(x, descending=True, stable=True)[1][:, 4])
    assert torch.equal(sample(x, u, top_p=torch.tensor([0.0, -1.0, -inf, 0.0, 0.0, 0.0], device="cuda")), top)
    assert torch.equal(sample(x, u, min_p=torch.tensor([1.0, 2.0, inf, 1.0, 1.0, 1.0], device="cuda")), top)
    assert torch.equal(sample(x, u, min_p=torch.full((6,), nan, device="cuda"), top_p=torch.full((6,), nan, device="cuda")), sample(x, u))
    # A very small temperature is the largest logit; an infinite one makes all tokens alike.
    assert torch.equal(sample(x, u, temperature=1e-30), top)
    flat = sample(x, torch.full((6,), 0.5, device="cuda"), temperature=torch.full((6,), inf, device="cuda"))
    assert torch.equal(flat, torch.sort(x, descending=True, stable=True)[1][:, 150])


@pytest.mark.parametrize("dtype", DTYPES)
def test_ruled_out_tokens(dtype):
    """-inf, NaN, the type's lowest value, +inf, both zeros; rows that nothing is left of."""
    inf, nan, low = float("inf"), float("nan"), torch.finfo(dtype).min
    rows = [[-inf] * 9, [nan] * 9, [-inf, nan, -inf, -3.0, -inf, nan, nan, nan, -inf], [low] * 9, [low, -inf, low, low, 1.0, low, nan, low, low],
            [0.0, -0.0, 0.0, -0.0, -inf, 0.0, -0.0, nan, -0.0], [inf, 1.0, inf, nan, -inf, 5.0, inf, 2.0, 3.0], [5.0] * 9,
            [-inf, -inf, -inf, -inf, -inf, -inf, -inf, -inf, 2.0]]
    x = torch.tensor(rows, dtype=dtype, device="cuda")
    for u in (0.0, 0.3, 0.5, 0.77, 0.9999):
        us = torch.full((len(rows),), u, device="cuda")
        for t, k, p, m in [(1.0, 0, 1.0, 0.0), (0.5, 3, 1.0, 0.0), (1.0, 0, 0.6, 0.0), (2.0, 0, 1.0, 0.5), (0.0, 0, 1.0, 0.0)]:
            compare(x, us, t, k, p, m)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("vocab", [9000, 60000, 151936])
def test_many_equal_logits(dtype, vocab):
    """A bin holds more tokens than are sorted: equal logits, few values, very high temperatures."""
    g = torch.Generator(device="cuda").manual_seed(vocab)
    few = torch.randint(0, 3, (6, vocab), generator=g, device="cuda").float()
    few[1] = 2.5
    few[2, : vocab // 2] = float("-inf")
    few[3] = torch.randn(vocab, generator=g, device="cuda") * 1e-3
    few[4] = torch.randn(vocab, generator=g, device="cuda") * 0.01 - 1000
    few[5, 17] = 9.0
    u = torch.tensor([0.31, 0.503, 0.77, 0.123, 0.9, 0.6], device="cuda")
    for t, k, p, m in [(1.0, 0, 1.0, 0.0), (1.0, 5000, 1.0, 0.0), (1.0, 0, 0.7, 0.0), (1.0, 7001, 0.45, 0.0), (50.0, 0, 1.0, 0.99), (1e4, 0, 0.3, 0.0),
                       (3.0, 4500, 0.95, 0.9), (1.0, 0, 1.0, 1.0)]:
        compare(few.to(dtype), u, t, k, p, m)


def test_rows_that_begin_anywhere():
    """Row strides and first elements off every 16-byte boundary, rows that end a tensor."""
    for dtype in DTYPES:
        flat = (torch.randn(7 * 1003 + 11, device="cuda") * 2).to(dtype)
        u = torch.rand(5, device="cuda")
        for first in range(9):
            x = flat[first:first + 7 * 1000].view(7, 1000)[2:, :997]
            assert torch.equal(sample(x, u, top_p=0.9), sample(x.contiguous(), u, top_p=0.9))
        tail = flat[-15:].view(5, 3)
        assert torch.equal(sample(tail, u), sample(tail.clone(), u))
        one = flat[:1000].view(1, 1000).expand(5, -1)
        assert torch.equal(sample(one, u), sample(one.contiguous(), u))


def test_draws_follow_the_distribution():
    """Evenly spaced numbers give each token its share: of 4096, the count is off by one at most for each end of its interval."""
    x = torch.tensor([[1.0, 3.0, -2.0, 2.5, 0.0, 3.0]], device="cuda").expand(4096, -1)
    u = (torch.arange(4096, device="cuda").float() + 0.5) / 4096
    counts = torch.bincount(sample(x, u, temperature=0.8), minlength=6).cpu().double()
    assert bool(((counts - 4096 * torch.softmax(x[0].double().cpu() / 0.8, 0)).abs() <= 1.0).all())


def test_no_rows():
    assert sample(torch.empty(0, 10, device="cuda"), torch.empty(0, device="cuda")).shape == (0,)


def test_results_in_a_given_tensor():
    x, u = inputs(4, 100, torch.float32)
    out = torch.zeros(4, dtype=torch.int64, device="cuda")
    assert sample(x, u, out=out) is out and torch.equal(out, sample(x, u))
