"""A cache whose tensors are replaced: every step uses the one that is there, and what does not fit is refused.

The tensors that were there stay alive, so that a step that used them still would read and write memory of the test's own."""
import copy

import pytest
import torch

from afterimage_amd.runtime.attention import rotary_tables, tree_attention
from afterimage_amd.runtime.kv_cache import PagedKVCache

pytestmark = pytest.mark.gpu

KINDS = [torch.bfloat16, torch.float8_e4m3fn]
NAMES = ["pool", "page_table", "lengths", "held", "refs", "status", "scales"]


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def filled(kind, seed):
    """A cache of two layers with 20 and 35 positions, and the tensors it was made of."""
    cache = PagedKVCache.allocate(2, 12, 16, 2, 64, 4, 5, kind)
    g = torch.Generator(device="cuda").manual_seed(seed)
    cache.pool.view(torch.uint8 if kind is torch.float8_e4m3fn else torch.int16).zero_()
    if cache.scales is not None:
        cache.scales.fill_(1.0)
    cache.reserve(ints([0, 2]), ints([20, 35]))
    for layer in range(2):
        k, v = (torch.randn(55, 2, 64, generator=g, device="cuda").bfloat16() for _ in range(2))
        cache.append(layer, k, v, ints([0, 2]), ints([0, 20, 55]))
    cache.advance(ints([0, 2]), ints([0, 20, 55]))
    cache.check()
    return cache


def names(kind):
    return NAMES if kind is torch.float8_e4m3fn else NAMES[:-1]


def plain(cache, layer, q):
    more = {} if cache.scales is None else {"k_scales": cache.scales[layer, 0], "v_scales": cache.scales[layer, 1]}
    return tree_attention(q, cache.pool[layer, 0], cache.pool[layer, 1], cache.page_table, cache.lengths, ints([0, 2]), ints([0, 1, 2]),
                          max_drafts=1, **more)


@pytest.mark.parametrize("kind", KINDS)
def test_attention_over_tensors_that_were_replaced(kind):
    """Of one cache after the other: its attention is what tree_attention gives over the tensors that are there."""
    cache, other = filled(kind, 1), filled(kind, 2)
    other.lengths.copy_(ints([3, 0, 30, 0]))
    other.page_table.copy_(other.page_table.flip(1).roll(-2, 1))
    old = [getattr(cache, name) for name in names(kind)]
    q = torch.randn(2, 4, 64, dtype=torch.bfloat16, device="cuda")
    last = cache.attend(1, q, ints([0, 2]), ints([0, 1, 2]), max_drafts=1)
    for name in ("lengths", "page_table", "pool", "scales")[:4 if kind is torch.float8_e4m3fn else 3]:
        setattr(cache, name, getattr(other, name).clone())
        for layer in range(2):
            got = cache.attend(layer, q, ints([0, 2]), ints([0, 1, 2]), max_drafts=1)
            assert torch.equal(got, plain(cache, layer, q)), name
        assert not torch.equal(got, last), name
        last = got
    assert len(old) == len(names(kind))


@pytest.mark.parametrize("kind", KINDS)
def test_every_step_uses_the_tensors_that_are_there(kind):
    """A cache over copies of its tensors, put in one by one, goes the way of one that was left alone; the originals stay."""
    cache, other = filled(kind, 3), filled(kind, 3)
    old = {name: getattr(cache, name) for name in names(kind)}
    for name in names(kind):
        setattr(cache, name, old[name].clone())
    before = {name: x.clone() for name, x in old.items()}
    cos, sin = rotary_tables(64, 64)
    g = torch.Generator(device="cuda").manual_seed(4)
    q, k, v = (torch.randn(5, h, 64, generator=g, device="cuda").bfloat16() for h in (4, 2, 2))
    for c in (cache, other):
        c.reserve(ints([0, 2]), ints([3, 2]))
        for layer in range(2):
            c.append_rotated(layer, q, k, v, ints([0, 2]), ints([0, 3, 5]), cos, sin)
        c.commit(ints([0, 2]), ints([[1, 2], [0, 0]]), ints([2, 1]))
        c.fork(ints([0, 2]), ints([1, 3]))
        c.release(ints([0]))
        c.compact()
        c.append(0, k, v, ints([44]), ints([0, 5]))  # no such slot
        assert int(c.status) == 4
    for name in names(kind):
        a, b = getattr(cache, name), getattr(other, name)
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8)), name
        assert torch.equal(old[name].view(torch.uint8), before[name].view(torch.uint8)), name
    got, want = (c.read(1, ints([1, 3]), ints([0, 22, 58]), 58) for c in (cache, other))
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.parametrize("kind", KINDS)
def test_tensors_that_do_not_fit_are_refused(kind):
    cache = filled(kind, 5)
    q = torch.randn(2, 4, 64, dtype=torch.bfloat16, device="cuda")
    want = cache.attend(0, q, ints([0, 2]), ints([0, 1, 2]), max_drafts=1)
    bad = [("pool", cache.pool[:1]), ("pool", cache.pool.view(torch.uint8)), ("pool", cache.pool.transpose(3, 4).contiguous().transpose(3, 4)),
           ("page_table", cache.page_table[:, :4]), ("page_table", cache.page_table.long()), ("lengths", cache.lengths.cpu()),
           ("lengths", torch.zeros(4, 2, dtype=torch.int32, device="cuda")[:, 0]), ("held", cache.held[:3]), ("refs", cache.refs.float()),
           ("status", ints([0, 0])), ("scales", torch.zeros(3, device="cuda")), ("lengths", None), ("pool", 7)]
    for name, x in bad:
        had = getattr(cache, name)
        with pytest.raises(ValueError, match=name):
            setattr(cache, name, x)
        assert getattr(cache, name) is had
    assert torch.equal(cache.attend(0, q, ints([0, 2]), ints([0, 1, 2]), max_drafts=1), want)


@pytest.mark.parametrize("kind", KINDS)
def test_a_copied_object_keeps_its_own_tensors(kind):
    cache = filled(kind, 6)
    other = copy.copy(cache)
    q = torch.randn(2, 4, 64, dtype=torch.bfloat16, device="cuda")
    want = [cache.attend(layer, q, ints([0, 2]), ints([0, 1, 2]), max_drafts=1) for layer in range(2)]
    held = cache.lengths
    other.lengths = ints([3, 0, 30, 0])
    other.pool = torch.zeros_like(cache.pool)
    for layer in range(2):
        assert torch.equal(cache.attend(layer, q, ints([0, 2]), ints([0, 1, 2]), max_drafts=1), want[layer])
        assert bool((other.attend(layer, q, ints([0, 2]), ints([0, 1, 2]), max_drafts=1) == 0).all())
    other.advance(ints([0]), ints([0, 1]))
    assert cache.lengths is held and held.tolist() == [20, 0, 35, 0] and other.lengths.tolist() == [4, 0, 30, 0]
