"""Pools, rows and logits whose offsets pass 32 bits."""
import pytest
import torch

from afterimage_amd.runtime.attention import rotary_tables
from afterimage_amd.runtime.kv_cache import PagedKVCache
from afterimage_amd.runtime.sampling import sample

pytestmark = pytest.mark.gpu


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("kind,n_pages", [(torch.float8_e4m3fn, 34000), (torch.bfloat16, 17000)])
def test_pages_past_four_gigabytes(kind, n_pages):
    """The same rows in pages at both ends of a pool of 4.2 GiB a plane give the same results."""
    kv, dim, page = 8, 128, 128
    cache = PagedKVCache.allocate(1, n_pages, page, kv, dim, 2, 3, kind)
    assert cache.pool[0, 0].numel() * cache.pool.element_size() > 1 << 32
    cache.page_table.copy_(ints([[0, 1, 2], [n_pages - 1, n_pages - 3, n_pages - 2]]))
    cache.held.fill_(3)
    cache.refs[[0, 1, 2, n_pages - 1, n_pages - 2, n_pages - 3]] = 1
    g = torch.Generator(device="cuda").manual_seed(0)
    tables = rotary_tables(400, dim)
    q, k, v = (torch.randn(300, h, dim, generator=g, device="cuda").bfloat16() for h in (16, kv, kv))
    q, k, v = (torch.cat((x, x)) for x in (q, k, v))
    slots, offsets = ints([0, 1]), ints([0, 300, 600])
    got = cache.append_rotated(0, q, k, v, slots, offsets, *tables)
    assert torch.equal(got[:300], got[300:])
    rows = cache.read(0, slots, offsets, 600)
    assert all(torch.equal(x[:300], x[300:]) for x in rows) and bool((rows[1][:300].float() - v[:300].float()).abs().max() < 0.5)
    cache.lengths.copy_(ints([290, 290]))
    last = torch.cat((got[290:300], got[590:]))
    o = cache.attend(0, last, slots, ints([0, 10, 20]), max_drafts=10, max_context=290)
    assert torch.equal(o[:10], o[10:]) and bool(torch.isfinite(o).all())
    cache.commit(slots, ints([[2, 5], [2, 5]]), ints([2, 2]))
    rows = cache.read(0, slots, ints([0, 292, 584]), 584)
    assert all(torch.equal(x[:292], x[292:]) for x in rows)
    cache.release(ints([0]))
    assert int(cache.compact()) == 3
    after = cache.read(0, ints([1]), ints([0, 292]), 292)
    assert all(torch.equal(x, y[292:]) for x, y in zip(after, rows))
    cache.check()


def test_logits_past_four_gigabytes():
    """16384 rows of 151936: the last ones as if they were alone."""
    x = torch.empty(16384, 151936, dtype=torch.bfloat16, device="cuda")
    x[-3:] = torch.randn(3, 151936, device="cuda") * 2
    x[:-3] = torch.randn(151936, device="cuda").bfloat16()
    u = torch.rand(16384, device="cuda")
    got = sample(x, u, top_p=0.9)
    assert torch.equal(got[-3:], sample(x[-3:].clone(), u[-3:], top_p=0.9))
    assert torch.equal(got[:5], sample(x[:5].clone(), u[:5], top_p=0.9))
