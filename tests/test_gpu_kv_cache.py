"""The paged cache's steps against a model of it in Python lists."""
import random

import pytest
import torch

from afterimage_amd.runtime.kv_cache import PagedKVCache

pytestmark = pytest.mark.gpu


def _ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


class Model:
    """What the cache holds: a list of rows (numbers that stand for a row's
    keys and values) and of pages for each slot."""

    def __init__(self, n_pages, page, max_seqs, max_pages):
        self.n_pages, self.page, self.max_pages = n_pages, page, max_pages
        self.rows = [[] for _ in range(max_seqs)]    # committed rows
        self.pages = [[] for _ in range(max_seqs)]

    def refs(self):
        r = [0] * self.n_pages
        for row in self.pages:
            for p in row:
                r[p] += 1
        return r

    def free(self):
        return [p for p, r in enumerate(self.refs()) if r == 0]

    def reserve(self, seqs, tokens):
        free = self.free()
        for s, n in zip(seqs, tokens):
            while len(self.pages[s]) * self.page < len(self.rows[s]) + n:
                self.pages[s].append(free.pop(0))

    def fork(self, src, dst):
        free = self.free()
        new = []
        for s, d in zip(src, dst):
            n = len(self.rows[s])
            pages = self.pages[s][:n // self.page]
            if s != d and n % self.page:
                pages = pages + [free.pop(0)]
            new.append((list(self.rows[s]), pages if s != d else self.pages[s]))
        for d, (rows, pages) in zip(dst, new):
            self.rows[d], self.pages[d] = rows, pages

    def release(self, seqs):
        for s in seqs:
            self.rows[s], self.pages[s] = [], []

    def compact(self):
        refs = self.refs()
        n = sum(r > 0 for r in refs)
        moves = dict(zip([p for p in range(n, self.n_pages) if refs[p]], [p for p in range(n) if not refs[p]]))
        self.pages = [[moves.get(p, p) for p in row] for row in self.pages]
        return n


class Pair:
    """The cache and its model, stepped together."""

    LAYERS, HEADS, DIM = 3, 2, 16

    def __init__(self, n_pages=40, page=4, max_seqs=7, max_pages=9, dtype=torch.bfloat16):
        self.cache = PagedKVCache.allocate(self.LAYERS, n_pages, page, self.HEADS, self.DIM, max_seqs, max_pages, dtype)
        self.cache.pool.fill_(-1.0)
        self.model = Model(n_pages, page, max_seqs, max_pages)
        self.next = 0

    def row(self, number, layer):
        """[keys or values, head, dim] of the row that a number stands for, exact in 16 bits."""
        base = torch.arange(2 * self.HEADS * self.DIM, device="cuda").view(2, self.HEADS, self.DIM)
        return ((base * 7 + number * 31 + layer * 5) % 251).to(self.cache.pool.dtype)

    def append(self, seqs, counts):
        """New rows for every layer; returns their numbers."""
        offsets = [sum(counts[:i]) for i in range(len(counts) + 1)]
        numbers = list(range(self.next, self.next + offsets[-1]))
        self.next += offsets[-1]
        for layer in range(self.LAYERS):
            if numbers:
                kv = torch.stack([self.row(x, layer) for x in numbers], 1)
                self.cache.append(layer, kv[0], kv[1], _ints(seqs), _ints(offsets))
        return [numbers[offsets[i]:offsets[i + 1]] for i in range(len(counts))], offsets

    def write(self, seqs, counts):
        self.cache.reserve(_ints(seqs), _ints(counts))
        self.model.reserve(seqs, counts)
        numbers, offsets = self.append(seqs, counts)
        self.cache.advance(_ints(seqs), _ints(offsets))
        for s, x in zip(seqs, numbers):
            self.model.rows[s] += x

    def draft(self, seqs, counts, accepted, new_lengths=None):
        self.cache.reserve(_ints(seqs), _ints(counts))
        self.model.reserve(seqs, counts)
        numbers, _ = self.append(seqs, counts)
        most = max(1, max(len(a) for a in accepted))
        paths = _ints([a + [0] * (most - len(a)) for a in accepted])
        self.cache.commit(_ints(seqs), paths, _ints([len(a) for a in accepted]), new_lengths)
        for s, x, a in zip(seqs, numbers, accepted):
            self.model.rows[s] += [x[i] for i in a]

    def fork(self, src, dst):
        self.cache.fork(_ints(src), _ints(dst))
        self.model.fork(src, dst)

    def release(self, seqs):
        self.cache.release(_ints(seqs))
        self.model.release(seqs)

    def compact(self):
        assert int(self.cache.compact()) == self.model.compact()

    def check(self):
        c, m = self.cache, self.model
        assert c.lengths.tolist() == [len(r) for r in m.rows]
        assert c.held.tolist() == [len(p) for p in m.pages]
        assert c.page_table.tolist() == [p + [-1] * (m.max_pages - len(p)) for p in m.pages]
        assert c.refs.tolist() == m.refs()
        c.check()
        for s, rows in enumerate(m.rows):
            for layer in range(self.LAYERS):
                if rows:
                    got = torch.stack([c.pool[layer, :, m.pages[s][j // m.page], :, j % m.page] for j in range(len(rows))])
                    assert torch.equal(got, torch.stack([self.row(x, layer) for x in rows])), (s, layer)


@pytest.mark.parametrize("free", [[12999], [4095, 4096, 8192, 12287], list(range(8190, 8200)), list(range(5)) + [9000, 9001], []])
def test_pools_of_several_scans(free):
    """More pages than a scan of them takes at a time, the free ones around its ends: the lowest are reserved and forked, or nothing is."""
    n = 13000
    c = PagedKVCache.allocate(1, n, 1, 1, 8, 4, 20)
    refs = torch.ones(n, dtype=torch.int32)
    refs[free] = 0
    c.refs.copy_(refs)
    more = len(free) // 2
    c.reserve(_ints([2, 0]), _ints([more, len(free) - more]))
    c.check()
    assert c.page_table[2, :more].tolist() == free[:more] and c.page_table[0, :len(free) - more].tolist() == free[more:]
    assert c.held.tolist() == [len(free) - more, 0, more, 0] and int(c.refs.min()) == 1
    before = c.page_table.clone()
    c.reserve(_ints([1, 3]), _ints([1, 0]))
    with pytest.raises(RuntimeError, match="too few"):
        c.check()
    assert torch.equal(c.page_table, before) and int(c.refs.max()) == 1


@pytest.mark.parametrize("free", [[12999], [0, 4096], list(range(4000, 4200)) + [12000], list(range(0, 13000, 3))])
def test_pools_of_several_scans_are_compacted(free):
    n = 13000
    c = PagedKVCache.allocate(1, n, 1, 1, 8, 2, 13000)
    in_use = sorted(set(range(n)) - set(free))
    refs = torch.zeros(n, dtype=torch.int32)
    refs[in_use] = torch.arange(1, len(in_use) + 1, dtype=torch.int32)
    c.refs.copy_(refs)
    c.page_table[1, :len(in_use)] = _ints(in_use)
    c.pool[0, :, :, 0, 0] = (torch.arange(n, device="cuda") % 251)[None, :, None].to(c.pool.dtype)
    assert int(c.compact()) == len(in_use)
    low = [p for p in free if p < len(in_use)]
    moves = dict(zip([p for p in in_use if p >= len(in_use)], low))
    assert c.page_table[1, :len(in_use)].tolist() == [moves.get(p, p) for p in in_use]
    where = torch.tensor([moves.get(p, p) for p in in_use])
    want = torch.zeros(n, dtype=torch.int32)
    want[where] = torch.arange(1, len(in_use) + 1, dtype=torch.int32)
    assert torch.equal(c.refs.cpu(), want)
    assert torch.equal(c.pool[0, 1, where.cuda(), 0, 0, 3].cpu(), (torch.tensor(in_use) % 251).to(c.pool.dtype))


def test_reserve_append_advance():
    p = Pair()
    p.write([0, 3], [5, 1])
    p.check()
    p.write([3, 1, 0], [3, 8, 0])
    p.check()
    p.write([1], [1])
    p.check()


def test_fork_shares_full_pages_and_copies_the_last():
    p = Pair()
    p.write([0, 1], [10, 8])
    p.fork([0, 0, 1], [2, 3, 4])
    p.check()
    p.write([0, 2, 3, 4], [1, 3, 6, 2])   # the branches go their own ways
    p.check()
    p.release([0])
    p.check()


def test_fork_reorders_beams():
    """Sources that are themselves replaced, kept slots, and slots that held more before."""
    p = Pair()
    p.write([0, 1, 2, 3], [10, 7, 13, 2])
    p.fork([1, 1, 0, 3], [0, 1, 2, 3])
    p.check()
    p.fork([3, 2, 1, 0], [0, 1, 2, 3])
    p.check()


def test_fork_does_not_pass_on_reserved_pages():
    p = Pair()
    p.write([0], [6])
    p.cache.reserve(_ints([0]), _ints([20]))
    p.model.reserve([0], [20])
    p.fork([0], [1])
    p.check()


def test_release_twice_in_a_call_and_of_an_empty_slot():
    p = Pair()
    p.write([0, 1], [10, 8])
    p.cache.release(_ints([0, 0, 5]))
    p.model.release([0])
    p.check()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("apart", [False, True])
def test_commit_moves_the_accepted_path(apart, dtype):
    p = Pair(dtype=dtype)
    p.write([0, 1, 2], [3, 8, 1])
    new = torch.full((7,), -9, dtype=torch.int32, device="cuda") if apart else None
    p.draft([2, 0, 1], [9, 12, 4], [[0, 2, 3, 8], [1, 4, 5, 6, 7, 11], []], new)
    if apart:
        assert new.tolist() == [9, 8, 5, -9, -9, -9, -9] and p.cache.lengths.tolist()[:3] == [3, 8, 1]
        p.cache.lengths[:3] = new[:3]
    p.check()


def test_commit_of_a_long_path():
    p = Pair(n_pages=80, page=4, max_seqs=2, max_pages=80)
    p.write([1], [5])
    p.draft([1], [300], [[i for i in range(300) if i % 7 != 2]])
    p.check()


def test_compact():
    p = Pair()
    p.write([0, 1, 2, 3], [10, 7, 13, 20])
    p.fork([0, 3], [4, 5])
    p.release([0, 1])
    p.compact()
    p.check()
    p.compact()   # nothing left to move
    p.check()
    p.release([2, 3, 4, 5])
    p.compact()
    p.check()


def test_compact_into_other_tensors():
    p = Pair()
    p.write([0, 1, 2], [10, 7, 13])
    p.release([0])
    before = p.cache.page_table.clone(), p.cache.refs.clone()
    table, refs = torch.zeros_like(before[0]), torch.zeros_like(before[1])
    used = p.cache.compact(new_table=table, new_refs=refs)
    assert torch.equal(p.cache.page_table, before[0]) and torch.equal(p.cache.refs, before[1])
    p.cache.page_table.copy_(table)
    p.cache.refs.copy_(refs)
    assert int(used) == p.model.compact()
    p.check()


@pytest.mark.parametrize("seed", range(6))
def test_many_steps(seed):
    rng = random.Random(seed)
    p = Pair(n_pages=60, page=rng.choice((1, 3, 4)), max_seqs=7, max_pages=30)
    for _ in range(25):
        seqs = rng.sample(range(7), rng.randint(1, 4))
        step = rng.choice(("write", "draft", "fork", "release", "compact"))
        room = 24 // p.model.page
        if step == "write":
            counts = [rng.randint(0, 4) if len(p.model.pages[s]) < room else 0 for s in seqs]
            if sum(counts) + len(seqs) < len(p.model.free()):
                p.write(seqs, counts)
        elif step == "draft":
            seqs = [s for s in seqs if len(p.model.pages[s]) < room] or seqs[:1]
            counts = [rng.randint(1, 5) for _ in seqs]
            if sum(counts) + len(seqs) < len(p.model.free()) and all(len(p.model.pages[s]) < room for s in seqs):
                p.draft(seqs, counts, [sorted(rng.sample(range(c), rng.randint(0, c))) for c in counts])
        elif step == "fork":
            src = [rng.randrange(7) for _ in seqs]
            if len(seqs) <= len(p.model.free()):
                p.fork(src, seqs)
        elif step == "release":
            p.release(seqs[:2])
        else:
            p.compact()
        p.check()


def test_too_few_pages_change_nothing():
    p = Pair(n_pages=6)
    p.write([0, 1], [10, 6])
    p.cache.reserve(_ints([0, 2]), _ints([1, 8]))     # 2 pages, 1 free
    with pytest.raises(RuntimeError, match="free pages"):
        p.cache.check()
    p.check()
    p.cache.fork(_ints([0, 0]), _ints([2, 3]))
    with pytest.raises(RuntimeError, match="free pages"):
        p.cache.check()
    p.check()
    p.fork([0], [2])
    p.check()


def test_what_does_not_exist_is_reported():
    p = Pair()
    p.write([0], [10])
    c = p.cache
    for step in (lambda: c.reserve(_ints([7]), _ints([1])), lambda: c.release(_ints([-1])), lambda: c.fork(_ints([0]), _ints([9])),
                 lambda: c.commit(_ints([70]), _ints([[0]]), _ints([1])), lambda: c.advance(_ints([7]), _ints([0, 0])),
                 lambda: c.reserve(_ints([1]), _ints([-1]))):
        step()
        with pytest.raises(RuntimeError, match="does not exist"):
            c.check()
        p.check()
    k = torch.zeros(3, p.HEADS, p.DIM, dtype=torch.bfloat16, device="cuda")
    for step in (lambda: c.reserve(_ints([0]), _ints([100])), lambda: c.advance(_ints([0]), _ints([0, 3])),
                 lambda: c.append(0, k, k, _ints([0]), _ints([0, 3])), lambda: c.commit(_ints([0]), _ints([[2]]), _ints([1]))):
        step()
        with pytest.raises(RuntimeError, match="past a sequence's pages"):
            c.check()
        # Rows that had a page were written past the length, where nothing is held yet.
        p.check()


def test_refusals():
    c = PagedKVCache.allocate(2, 8, 4, 2, 16, 3, 4)
    k = torch.zeros(2, 2, 16, dtype=torch.bfloat16, device="cuda")
    one, at = _ints([0]), _ints([0, 2])
    for step, message in [
        (lambda: c.append(2, k, k, one, at), "layer"), (lambda: c.append(0, k.half(), k, one, at), "k must be"),
        (lambda: c.append(0, k, k[:1], one, at), "one shape"), (lambda: c.append(0, k, k, one, _ints([0])), "offsets"),
        (lambda: c.append(0, k.transpose(1, 2).contiguous().transpose(1, 2), k, one, at), "last dimension"),
        (lambda: c.reserve(one.long(), one), "seqs"), (lambda: c.reserve(one, _ints([1, 2])), "tokens"),
        (lambda: c.fork(one, _ints([1, 2])), "dst"), (lambda: c.commit(one, _ints([0]), one), "accepted"),
        (lambda: c.commit(one, _ints([[0]]), one, new_lengths=_ints([0])), "new_lengths"),
        (lambda: c.compact(new_table=_ints([[0]])), "new_table"), (lambda: c.release(_ints([0] * 8193)), "at most 8192"),
        (lambda: PagedKVCache.allocate(2, 8, 4, 2, 12, 3, 4), "multiple of 8"),
        (lambda: PagedKVCache(c.pool[:, :1], c.page_table, c.lengths, c.held, c.refs, c.status), "pool"),
    ]:
        with pytest.raises(ValueError, match=message):
            step()
    with pytest.raises(RuntimeError, match="GPU only"):
        PagedKVCache.allocate(2, 8, 4, 2, 16, 3, 4, device="cpu")


def test_steps_replayed_from_a_graph():
    """Reserve, append, attend and commit in one graph, replayed with new inputs and no word from the host."""
    p = Pair(n_pages=60, page=4, max_seqs=3, max_pages=20)
    p.write([0, 1], [6, 11])
    c = p.cache
    seqs, offsets, tokens = _ints([0, 1]), _ints([0, 3, 6]), _ints([3, 3])
    rows = torch.zeros(p.LAYERS, 2, 6, p.HEADS, p.DIM, dtype=torch.bfloat16, device="cuda")
    q = torch.randn(6, 4, p.DIM, device="cuda").to(torch.bfloat16)
    masks = torch.tensor([[1], [3], [5]] * 2, dtype=torch.int64, device="cuda")
    paths, counts = _ints([[0, 2], [0, 1]]), _ints([2, 1])
    outs = [torch.zeros_like(q) for _ in range(p.LAYERS)]

    def step():
        c.reserve(seqs, tokens)
        for layer in range(p.LAYERS):
            c.append(layer, rows[layer, 0], rows[layer, 1], seqs, offsets)
            c.attend(layer, q, seqs, offsets, masks, max_drafts=3, out=outs[layer])
        c.commit(seqs, paths, counts)

    saved = [x.clone() for x in (c.pool, c.page_table, c.lengths, c.held, c.refs)]
    step()
    torch.cuda.synchronize()
    for x, y in zip((c.pool, c.page_table, c.lengths, c.held, c.refs), saved):
        x.copy_(y)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for _ in range(5):
        numbers = [list(range(p.next, p.next + 3)), list(range(p.next + 3, p.next + 6))]
        p.next += 6
        for layer in range(p.LAYERS):
            rows[layer] = torch.stack([p.row(x, layer) for x in numbers[0] + numbers[1]], 1)
        # The same steps, eagerly, on a copy of the cache.
        copy = PagedKVCache(*(x.clone() for x in (c.pool, c.page_table, c.lengths, c.held, c.refs, c.status)))
        copy.reserve(seqs, tokens)
        for layer in range(p.LAYERS):
            copy.append(layer, rows[layer, 0], rows[layer, 1], seqs, offsets)
        eager = [copy.attend(layer, q, seqs, offsets, masks, max_drafts=3) for layer in range(p.LAYERS)]
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(outs, eager))
        p.model.reserve([0, 1], [3, 3])
        p.model.rows[0] += [numbers[0][0], numbers[0][2]]
        p.model.rows[1] += [numbers[1][0]]
        p.check()


def test_another_stream():
    p = Pair()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        p.write([0, 1], [10, 8])
        p.fork([0], [2])
        p.draft([2, 1], [4, 4], [[0, 3], [1]])
        p.release([0])
        p.compact()
        p.check()
