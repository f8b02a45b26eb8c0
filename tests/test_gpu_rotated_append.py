"""Rows turned by their positions on their way into a cache, against products
and sums that are each rounded to fp32 (as the kernel's are: no tolerance)."""
import pytest
import torch

from afterimage_amd.runtime.attention import rotary_tables
from afterimage_amd.runtime.kv_cache import PagedKVCache
from tests.eight_bits import Copy, turn

pytestmark = pytest.mark.gpu

KINDS = [torch.bfloat16, torch.float16, torch.float8_e4m3fn]


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def make(kind, layers=2, n_pages=24, page=16, heads=2, dim=64, slots=4, most=6):
    cache = PagedKVCache.allocate(layers, n_pages, page, heads, dim, slots, most, kind)
    cache.pool.view(torch.uint8 if kind is torch.float8_e4m3fn else torch.int16).zero_()
    if cache.scales is not None:
        cache.scales.fill_(1.0)
    return cache


def step(cache, dtype, heads, half, interleaved, slots, lengths, sizes, positions=None, layer=1, seed=0, change=lambda q, k, v: (q, k, v), tables=None):
    """One call on both sides; returns the turned queries and what they should be."""
    g = torch.Generator().manual_seed(seed)
    n, kv, dim = sum(sizes), cache.kv_heads, cache.dim
    q, k, v = (torch.randn(n, h, dim, generator=g).to(dtype) for h in (heads, kv, kv))
    cos, sin = tables or rotary_tables(200, 2 * half, 1e4, "cpu")
    cache.reserve(ints(slots), ints(lengths))
    cache.lengths[torch.tensor(slots)] = ints(lengths)
    cache.reserve(ints(slots), ints(sizes))
    copy = Copy(cache)
    offsets = [sum(sizes[:i]) for i in range(len(sizes) + 1)]
    at = [lengths[b] + i for b, m in enumerate(sizes) for i in range(m)] if positions is None else positions
    tq, tk = (turn(x.float(), cos[at], sin[at], interleaved) for x in (q, k))
    for b, slot in enumerate(slots):
        for which, x in ((0, tk), (1, v.float())):
            for head in range(kv):
                part = x[offsets[b]:offsets[b + 1], head].double()
                if len(part):
                    copy.put(layer, which, head, slot, lengths[b], list(part))
    dq, dk, dv = change(q.cuda(), k.cuda(), v.cuda())
    got = cache.append_rotated(layer, dq, dk, dv, ints(slots), ints(offsets), cos.cuda(), sin.cuda(), None if positions is None else ints(positions),
                               interleaved=interleaved)
    cache.check()
    copy.same(cache)
    return got, tq.to(dtype)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dim,half", [(64, 32), (128, 64), (96, 48), (128, 16), (80, 40), (16, 8), (64, 12), (48, 3), (256, 128), (208, 100), (32, 1)])
def test_rows_turn(kind, interleaved, dim, half):
    dtype = torch.bfloat16 if kind is torch.float8_e4m3fn else kind
    cache = make(kind, dim=dim)
    got, want = step(cache, dtype, 6, half, interleaved, [2, 0, 3], [5, 0, 31], [1, 20, 4], seed=dim + half)
    assert torch.equal(got.cpu(), want)


@pytest.mark.parametrize("dim", [8, 24, 40, 72, 136])
def test_dims_of_eight_in_sixteen_bits(dim):
    cache = make(torch.bfloat16, dim=dim)
    for interleaved in (False, True):
        got, want = step(cache, torch.bfloat16, 3, dim // 2, interleaved, [1], [3], [9], seed=dim)
        assert torch.equal(got.cpu(), want)


@pytest.mark.parametrize("kind", KINDS)
def test_half_precision_queries_and_given_positions(kind):
    """Drafted trees: several rows of one position. fp16 rows go into a cache of 8 bits too."""
    dtype = torch.float16 if kind is torch.float8_e4m3fn else kind
    cache = make(kind)
    positions = [9, 10, 10, 11, 11, 199, 0]
    got, want = step(cache, dtype, 4, 32, False, [3, 1], [9, 2], [5, 2], positions)
    assert torch.equal(got.cpu(), want)


@pytest.mark.parametrize("kind", [torch.bfloat16, torch.float8_e4m3fn])
@pytest.mark.parametrize("interleaved,half", [(False, 32), (True, 32), (False, 12)])
def test_strides_and_the_queries_own_memory(kind, interleaved, half):
    """Queries, keys and values of one product's output, and the result in their place."""
    cache = make(kind)

    def packed(q, k, v):
        both = torch.cat((q, k, v), 1)
        return both[:, :4], both[:, 4:6], both[:, 6:]

    got, want = step(cache, torch.bfloat16, 4, half, interleaved, [0, 2], [17, 3], [6, 30], change=packed)
    assert torch.equal(got.cpu(), want)
    q = torch.randn(36, 4, 64, dtype=torch.bfloat16, device="cuda")
    wide = torch.randn(36, 9, 64, dtype=torch.bfloat16, device="cuda")
    wide[:, 3:7] = q
    k = torch.randn(36, 2, 64, dtype=torch.bfloat16, device="cuda")
    cos, sin = rotary_tables(64, 2 * half)
    offsets, slots = ints([0, 6, 36]), ints([0, 2])
    apart = cache.append_rotated(0, q, k, k, slots, offsets, cos, sin, interleaved=interleaved)
    rest = wide.clone()
    same = cache.append_rotated(0, wide[:, 3:7], k, k, slots, offsets, cos, sin, interleaved=interleaved, out=wide[:, 3:7])
    assert torch.equal(apart, same) and torch.equal(wide[:, :3], rest[:, :3]) and torch.equal(wide[:, 7:], rest[:, 7:])


@pytest.mark.parametrize("kind", [torch.bfloat16, torch.float8_e4m3fn])
def test_tables_that_begin_anywhere(kind):
    """Tables off a 16-byte boundary give the same bits."""
    cos, sin = (torch.cat((torch.zeros(1), x.flatten())).cuda()[1:].view(x.shape) for x in rotary_tables(200, 64, 1e4, "cpu"))
    cache, other = make(kind), make(kind)
    q, k = (torch.randn(7, h, 64, dtype=torch.bfloat16, device="cuda") for h in (4, 2))
    for c in (cache, other):
        c.reserve(ints([0]), ints([7]))
    a = cache.append_rotated(0, q, k, k, ints([0]), ints([0, 7]), cos, sin)
    b = other.append_rotated(0, q, k, k, ints([0]), ints([0, 7]), cos.clone(), sin.clone())
    assert torch.equal(a, b) and torch.equal(cache.pool[0].view(torch.uint8), other.pool[0].view(torch.uint8))


@pytest.mark.parametrize("kind", [torch.bfloat16, torch.float8_e4m3fn])
def test_rows_that_are_left_out(kind):
    """Rows of no sequence, of no slot, of positions past the tables, of no page: queries stay as they were, keys too."""
    cache = make(kind, layers=1)
    cache.reserve(ints([0]), ints([16]))
    cos, sin = rotary_tables(8, 64)
    q, k = (torch.randn(12, h, 64, dtype=torch.bfloat16, device="cuda") for h in (4, 2))
    out = torch.full_like(q, 5.0)
    cache.append_rotated(0, q, k, k, ints([0]), ints([2, 6]), cos, sin, out=out)
    cache.check()
    assert bool((out[:2] == 5.0).all()) and bool((out[6:] == 5.0).all()) and not bool((out[2:6] == 5.0).any(-1).all())
    assert torch.equal(out[2], q[2])  # position 0
    out.fill_(5.0)
    cache.append_rotated(0, q, k, k, ints([0]), ints([0, 12]), cos, sin, out=out)  # positions 8 .. 11 have no angles
    with pytest.raises(RuntimeError, match="does not exist"):
        cache.check()
    assert bool((out[8:] == 5.0).all()) and not bool((out[:8] == 5.0).any(-1).all())
    for positions in ([-1] * 12, [8] * 12, [2 ** 31 - 1] * 12):
        out.fill_(5.0)
        before = cache.pool.view(torch.uint8).clone()
        cache.append_rotated(0, q, k, k, ints([0]), ints([0, 12]), cos, sin, ints(positions), out=out)
        with pytest.raises(RuntimeError, match="does not exist"):
            cache.check()
        assert bool((out == 5.0).all()) and torch.equal(cache.pool.view(torch.uint8), before)
    out.fill_(5.0)
    cache.append_rotated(0, q, k, k, ints([44]), ints([0, 12]), cos, sin, out=out)
    with pytest.raises(RuntimeError, match="does not exist"):
        cache.check()
    assert bool((out == 5.0).all())
    # No room: the queries turn all the same.
    cache.append_rotated(0, q[:4], k[:4], k[:4], ints([1]), ints([0, 4]), cos, sin, out=out[:4])
    with pytest.raises(RuntimeError, match="past a sequence's pages"):
        cache.check()
    assert torch.equal(out[0], q[0])


def test_tables_of_far_positions():
    """Angles are taken in 64 bits: a table's entry is off by half a step of fp32 (and 2^-50 of the angle)."""
    cos, sin = rotary_tables(1 << 18, 16, 5e5)
    p = (1 << 18) - 1
    for i in range(8):
        angle = torch.tensor(p, dtype=torch.float64) * torch.tensor(5e5, dtype=torch.float64) ** (-2 * i / 16)
        assert abs(float(cos[p, i]) - float(angle.cos())) <= 2.0 ** -25 + p * 2.0 ** -50
        assert abs(float(sin[p, i]) - float(angle.sin())) <= 2.0 ** -25 + p * 2.0 ** -50
