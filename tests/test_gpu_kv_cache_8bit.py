"""The paged cache in 8 bits against its definition: every code and scale of the
pool, so that what a step must leave alone is looked at too."""
import pytest
import torch

from afterimage_amd.runtime.kv_cache import PagedKVCache
from tests.eight_bits import Copy

pytestmark = pytest.mark.gpu


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def make(layers=2, n_pages=24, page=32, heads=2, dim=48, slots=5, most=6, seed=0):
    """An empty cache whose pool and scales hold values that nothing has put there."""
    g = torch.Generator().manual_seed(seed)
    cache = PagedKVCache.allocate(layers, n_pages, page, heads, dim, slots, most, torch.float8_e4m3fn)
    cache.pool.copy_((torch.randn(cache.pool.shape, generator=g) * 40).clamp(-400, 400).to(torch.float8_e4m3fn))
    cache.scales.copy_(torch.exp2(torch.randint(-9, 4, cache.scales.shape, generator=g).float()))
    return cache


def rows(g, n, heads, dim, dtype=torch.bfloat16, spread=12):
    """Rows of sizes that differ by many powers of two."""
    x = torch.randn(n, heads, dim, generator=g) * torch.exp2(torch.randint(-spread, spread // 2, (n, heads, 1), generator=g).float())
    return x.to(dtype)


def put(cache, copy, layer, k, v, slots, sizes):
    """append on both sides."""
    offsets = [sum(sizes[:i]) for i in range(len(sizes) + 1)]
    cache.append(layer, k.cuda(), v.cuda(), ints(slots), ints(offsets))
    for b, slot in enumerate(slots):
        for which, x in ((0, k), (1, v)):
            for head in range(cache.kv_heads):
                part = x[offsets[b]:offsets[b + 1], head].double()
                if len(part):
                    copy.put(layer, which, head, slot, int(copy.lengths[slot]), list(part))
    return offsets


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("page,dim,heads", [(16, 16, 1), (32, 48, 2), (16, 64, 3), (48, 96, 1), (64, 128, 2), (16, 256, 1), (32, 208, 2)])
def test_appends_form_blocks(dtype, page, dim, heads):
    cache = make(page=page, dim=dim, heads=heads, n_pages=30, most=-(-120 // page), seed=page + dim)
    g = torch.Generator().manual_seed(dim)
    copy = Copy(cache)
    # Whole blocks, blocks that grow a row at a time, none, and rows that end inside a block.
    for sizes in ([1, 16, 0], [1, 3, 17], [15, 1, 5], [30, 33, 1]):
        slots = [3, 0, 2]
        cache.reserve(ints(slots), ints(sizes))
        copy.table = cache.page_table.cpu().clone()
        n = sum(sizes)
        for layer in (1, 0):
            k, v = rows(g, n, heads, dim, dtype), rows(g, n, heads, dim, dtype)
            offsets = put(cache, copy, layer, k, v, slots, sizes)
        cache.advance(ints(slots), ints(offsets))
        for s, n in zip(slots, sizes):
            copy.lengths[s] += n
        copy.same(cache)
    cache.check()


def test_extremes_of_a_block():
    """Zeros, the largest and smallest numbers, infinities and NaN, alone and among others."""
    cache = make(layers=1, page=16, dim=16, heads=1, n_pages=12, slots=1, most=12)
    copy = Copy(cache)
    inf, nan = float("inf"), float("nan")
    big = torch.finfo(torch.bfloat16).max
    blocks = [[0.0], [big], [-big, 1.0], [2.0 ** -133], [2.0 ** -108, -2.0 ** -109], [inf], [nan, 3.0], [-inf, 448.0], [449.0, 2.0 ** -3],
              [464.0, 2.0 ** -9], [1.75, 1.7578125]]
    x = torch.zeros(16 * len(blocks), 1, 16)
    for i, b in enumerate(blocks):
        x[16 * i + 3, 0, :len(b)] = torch.tensor(b)
        x[16 * i + 9, 0, 2:2 + len(b)] = torch.tensor(b) / 2 if b[0] != big else torch.tensor(b)
    x = x.to(torch.bfloat16)
    cache.reserve(ints([0]), ints([len(x)]))
    copy.table = cache.page_table.cpu().clone()
    put(cache, copy, 0, x, -x, [0], [len(x)])
    copy.same(cache)
    cache.check()


def test_a_block_is_formed_anew_from_what_it_stands_for():
    """A row that raises a block's scale, one that was drafted and not kept, and the same rows twice."""
    cache = make(layers=1, page=16, dim=32, heads=1, n_pages=6, slots=2, most=3)
    copy = Copy(cache)
    g = torch.Generator().manual_seed(3)
    cache.reserve(ints([1]), ints([40]))
    copy.table = cache.page_table.cpu().clone()
    small, large = rows(g, 5, 1, 32, spread=4), rows(g, 3, 1, 32, spread=4) * 4096
    put(cache, copy, 0, small, small, [1], [5])
    cache.advance(ints([1]), ints([0, 5]))
    copy.lengths[1] = 5
    for x in (large, large, small):  # drafted, drafted again, replaced by small rows: the scale falls again
        put(cache, copy, 0, x, -x, [1], [len(x)])
        copy.same(cache)
    cache.check()


@pytest.mark.parametrize("page,dim", [(16, 64), (32, 128), (64, 256)])
def test_commits(page, dim):
    cache = make(layers=2, page=page, dim=dim, heads=2, n_pages=30, slots=6, most=8, seed=dim)
    copy = Copy(cache)
    g = torch.Generator().manual_seed(page)
    slots, lengths, drafts = [4, 1, 0, 5, 2], [7, 16, 0, 37, 15], 40
    paths = [[0, 1, 2, 3], [1, 2, 7, 8, 9, 21, 22, 23, 24, 25, 26, 27, 28, 29, 30, 31, 32, 39], [0, 3], [], [0, 2, 39]]
    cache.reserve(ints(slots), ints([n + drafts for n in lengths]))
    copy.table = cache.page_table.cpu().clone()
    for sizes, move in ((lengths, True), ([drafts] * 5, False)):
        for layer in range(2):
            k, v = rows(g, sum(sizes), 2, dim), rows(g, sum(sizes), 2, dim)
            offsets = put(cache, copy, layer, k, v, slots, sizes)
        if move:
            cache.advance(ints(slots), ints(offsets))
            for s, n in zip(slots, sizes):
                copy.lengths[s] += n
    copy.same(cache)
    most = max(map(len, paths))
    elsewhere = torch.full_like(cache.lengths, -7)
    cache.commit(ints(slots), ints([p + [0] * (most - len(p)) for p in paths]), ints([len(p) for p in paths]), elsewhere)
    want = cache.lengths.clone()
    for s, p in zip(slots, paths):
        copy.commit(s, p)
        want[s] += len(p)
    assert elsewhere.tolist() == [-7 if s not in slots else int(want[s]) for s in range(6)]
    cache.lengths.copy_(want)
    copy.same(cache)
    cache.check()


def test_commit_leaves_blocks_of_bad_pages_and_reports():
    cache = make(layers=1, page=16, dim=32, heads=1, n_pages=8, slots=2, most=4)
    cache.reserve(ints([0, 1]), ints([40, 40]))
    cache.page_table[0, 1] = 99
    before, scales = cache.pool.clone(), cache.scales.clone()
    cache.commit(ints([0]), ints([[3, 20]]), ints([2]))
    assert torch.equal(cache.pool.view(torch.uint8), before.view(torch.uint8)) and torch.equal(cache.scales, scales)
    with pytest.raises(RuntimeError, match="does not exist"):
        cache.check()
    for counts, text in (([3], "does not exist"), ([-1], "does not exist")):
        cache.commit(ints([1]), ints([[1, 2]]), ints(counts))
        with pytest.raises(RuntimeError, match=text):
            cache.check()
    assert torch.equal(cache.pool.view(torch.uint8), before.view(torch.uint8))


def test_forks_share_pages_and_copy_tails_with_their_scales():
    cache = make(layers=3, page=48, dim=32, heads=2, n_pages=20, slots=5, most=4)
    copy = Copy(cache)
    g = torch.Generator().manual_seed(8)
    sizes = [50, 96, 17]
    cache.reserve(ints([0, 1, 2]), ints(sizes))
    copy.table = cache.page_table.cpu().clone()
    for layer in range(3):
        offsets = put(cache, copy, layer, rows(g, sum(sizes), 2, 32), rows(g, sum(sizes), 2, 32), [0, 1, 2], sizes)
    cache.advance(ints([0, 1, 2]), ints(offsets))
    cache.fork(ints([0, 1, 2, 0]), ints([3, 4, 1, 0]))
    cache.check()
    assert cache.lengths.tolist() == [50, 17, 17, 50, 96] and cache.held.tolist() == [2, 1, 1, 2, 2]
    for layer in range(3):
        for which in range(2):
            for a, b, n in ((0, 3, 50), (2, 1, 17)):
                got, had = (cache.read(layer, ints([s]), ints([0, n]), n) for s in (b, a))
                assert torch.equal(got[which].nan_to_num(), had[which].nan_to_num())
                want = torch.stack([torch.stack([copy.row(layer, which, h, a, j) for h in range(2)]) for j in range(n)])
                assert torch.equal(got[which].cpu().double(), want)
    # A branch's rows change nothing of its source.
    before = cache.read(0, ints([0]), ints([0, 50]), 50)[0]
    x = rows(g, 9, 2, 32).cuda() * 1000
    cache.append(0, x, x, ints([3]), ints([0, 9]))
    assert torch.equal(cache.read(0, ints([0]), ints([0, 50]), 50)[0], before)
    # Then everything moves to the front.
    held = [cache.read(layer, ints([s]), ints([0, n]), n) for layer in range(3) for s, n in enumerate([50, 17, 17, 50, 96])]
    cache.release(ints([0]))
    used = int(cache.compact())
    assert used == int((cache.refs > 0).sum()) and bool((cache.refs[:used] > 0).all())
    after = [cache.read(layer, ints([s]), ints([0, n]), n) for layer in range(3) for s, n in enumerate([50, 17, 17, 50, 96]) if s]
    kept = [x for i, x in enumerate(held) if i % 5]
    assert all(torch.equal(a, b) for x, y in zip(kept, after) for a, b in zip(x, y))
    cache.check()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float8_e4m3fn])
def test_reads(dtype):
    """Any positions of any slots, past a length too; rows of no sequence and of no page stay as they were."""
    cache = make(page=32, dim=64, heads=3, n_pages=20, slots=4, most=5) if dtype is torch.float8_e4m3fn else \
        PagedKVCache.allocate(2, 20, 32, 3, 64, 4, 5, dtype)
    if dtype is not torch.float8_e4m3fn:
        cache.pool.normal_()
    cache.reserve(ints([0, 2, 3]), ints([100, 33, 32]))
    copy = Copy(cache)
    kinds = (torch.bfloat16, torch.float16) if dtype is torch.float8_e4m3fn else (dtype,)
    for kind in kinds:
        for starts in (None, [30, 0, 5]):
            k, v = (torch.full((80, 3, 64), 7.0, dtype=kind, device="cuda") for _ in range(2))
            offsets, slots = [2, 60, 60, 77], [0, 2, 3]
            cache.read(1, ints(slots), ints(offsets), 80, None if starts is None else ints(starts), dtype=kind, out=(k, v))
            for which, got in ((0, k), (1, v)):
                want = torch.full((80, 3, 64), 7.0, dtype=torch.float64)
                for b, slot in enumerate(slots):
                    for i in range(offsets[b], offsets[b + 1]):
                        at = i - offsets[b] + (starts[b] if starts else 0)
                        want[i] = torch.stack([copy.row(1, which, h, slot, at).double() for h in range(3)])
                assert torch.equal(got.cpu().double(), want.to(kind).double())
    cache.check()
    out = tuple(torch.full((6, 3, 64), 7.0, dtype=kinds[0], device="cuda") for _ in range(2))
    cache.read(0, ints([2, 9, 1]), ints([0, 3, 5, 6]), 6, ints([62, 0, 0]), dtype=kinds[0], out=out)  # past its pages, no slot, no pages
    assert bool((out[0][2:] == 7.0).all()) and not bool((out[0][:2] == 7.0).all())
    with pytest.raises(RuntimeError):
        cache.check()
    cache.read(0, ints([0]), ints([0, 2]), 2, ints([-1]), dtype=kinds[0])
    with pytest.raises(RuntimeError):
        cache.check()


def test_appends_report_what_cannot_be():
    cache = make(layers=1, page=16, dim=16, heads=1, n_pages=4, slots=2, most=4)
    cache.reserve(ints([0]), ints([20]))
    before, scales = cache.pool.view(torch.uint8).clone(), cache.scales.clone()
    x = torch.ones(40, 1, 16, dtype=torch.bfloat16, device="cuda")
    for slots, offsets, text in (([7], [0, 3], "does not exist"), ([-1], [0, 3], "does not exist"), ([1], [0, 3], "past a sequence's pages")):
        cache.append(0, x, x, ints(slots), ints(offsets))
        with pytest.raises(RuntimeError, match=text):
            cache.check()
    assert torch.equal(cache.pool.view(torch.uint8), before) and torch.equal(cache.scales, scales)
    # Rows past the pages are left out, those before them are not.
    cache.append(0, x, x, ints([0]), ints([0, 40]))
    with pytest.raises(RuntimeError, match="past a sequence's pages"):
        cache.check()
    assert bool((cache.read(0, ints([0]), ints([0, 32]), 32)[0] == 1.0).all())
    # Offsets that are no offsets.
    for offsets in ([5, 3], [-4, 2], [38, 90], [-9, -2]):
        cache.append(0, x, x, ints([0]), ints(offsets))
    torch.cuda.synchronize()
