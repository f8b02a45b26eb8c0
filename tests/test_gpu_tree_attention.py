"""Attention of drafted trees over a paged cache against its definition in 64 bits."""
import random

import pytest
import torch

from afterimage_amd.runtime.attention import tree_attention, tree_masks
from tests.attention_oracle import attend, check

pytestmark = pytest.mark.gpu


def _ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


class Case:
    """contexts[b] cached positions and drafts[b] drafted tokens for each
    sequence, slots and pages in no order; what no position holds is NaN."""

    def __init__(self, contexts, drafts, heads, kv, dim, page, dtype, seed=0, spare_slots=3):
        rng = random.Random(seed)
        g = torch.Generator(device="cuda").manual_seed(seed)
        self.contexts, self.drafts, self.heads, self.kv, self.dim, self.page, self.dtype = contexts, drafts, heads, kv, dim, page, dtype
        n = len(contexts)
        held = [-(-(c + d) // page) for c, d in zip(contexts, drafts)]
        self.n_pages = sum(held) + 5
        order = list(range(self.n_pages))
        rng.shuffle(order)
        slots = list(range(n + spare_slots))
        rng.shuffle(slots)
        self.slots = slots[:n]
        table = [[-1] * (max(held, default=0) + 1) for _ in range(n + spare_slots)]
        lengths = [0] * (n + spare_slots)
        shape = (self.n_pages, kv, page, dim)
        self.k = torch.full(shape, float("nan"), device="cuda", dtype=dtype)
        self.v = torch.full(shape, float("nan"), device="cuda", dtype=dtype)
        self.rows = []
        at = 0
        for b in range(n):
            pages = order[at:at + held[b]]
            at += held[b]
            table[self.slots[b]][:held[b]] = pages
            lengths[self.slots[b]] = contexts[b]
            m = contexts[b] + drafts[b]
            k, v = (torch.randn(m, kv, dim, generator=g, device="cuda").to(dtype) for _ in range(2))
            self.rows.append((k, v))
            for i, p in enumerate(pages):
                part = slice(i * page, min(m, (i + 1) * page))
                self.k[p, :, :part.stop - part.start] = k[part].transpose(0, 1)
                self.v[p, :, :part.stop - part.start] = v[part].transpose(0, 1)
        self.table, self.lengths, self.seqs = _ints(table), _ints(lengths), _ints(self.slots)
        self.offsets = _ints([sum(drafts[:b]) for b in range(n + 1)])
        self.q = (torch.randn(sum(drafts), heads, dim, generator=g, device="cuda") * 2).to(dtype)
        self.parents = [rng.randint(-1, t - 1) for d in drafts for t in range(d)]
        self.sees = []  # drafted tokens that each row sees
        for b, d in enumerate(drafts):
            first = sum(drafts[:b])
            for t in range(d):
                up = self.parents[first + t]
                self.sees.append({t} | (self.sees[first + up] if up >= 0 else set()))

    def bits(self, words=None):
        words = words or -(-max(self.drafts) // 64)
        out = []
        for seen in self.sees:
            m = sum(1 << j for j in seen)
            out.append([((m >> 64 * w & (1 << 64) - 1) ^ 1 << 63) - (1 << 63) for w in range(words)])
        return torch.tensor(out, dtype=torch.int64, device="cuda")

    def expected(self, scale=None):
        scale = self.dim ** -0.5 if scale is None else scale
        outs = []
        for b, (c, d) in enumerate(zip(self.contexts, self.drafts)):
            first = sum(self.drafts[:b])
            visible = torch.zeros(d, c + d, dtype=torch.bool)
            visible[:, :c] = True
            for t in range(d):
                for j in self.sees[first + t]:
                    visible[t, c + j] = True
            outs.append(attend(self.q[first:first + d], *self.rows[b], visible.cuda(), scale))
        return tuple(torch.cat(x) for x in zip(*outs))

    def run(self, masks="bits", **more):
        args = dict(q=self.q, k_pages=self.k, v_pages=self.v, page_table=self.table, lengths=self.lengths, seqs=self.seqs,
                    draft_offsets=self.offsets, masks=self.bits() if isinstance(masks, str) else masks, max_drafts=max(self.drafts))
        return tree_attention(**(args | more))


SHAPES = [
    # contexts, drafts, heads, kv_heads, dim, page
    ([1], [1], 1, 1, 64, 16),
    ([0], [1], 4, 2, 128, 16),
    ([31, 32, 33], [1, 1, 1], 40, 8, 128, 16),
    ([500, 7, 64], [3, 6, 1], 40, 8, 128, 32),
    ([500, 0, 127, 128], [12, 5, 1, 8], 40, 8, 128, 64),
    ([900, 300], [33, 13], 40, 8, 128, 16),
    ([200, 130], [64, 3], 16, 2, 64, 64),
    ([100, 1000], [70, 130], 8, 1, 64, 5),
    ([77, 300], [6, 2], 6, 3, 96, 1),
    ([200, 50], [2, 9], 8, 4, 256, 48),
    ([700, 50], [40, 9], 8, 4, 256, 32),
    ([260], [7], 12, 4, 8, 24),
    ([3000, 4100, 5], [4, 1, 2], 16, 16, 64, 128),
    ([6000, 9000], [5, 16], 40, 8, 128, 128),
]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("contexts,drafts,heads,kv,dim,page", SHAPES)
def test_trees(contexts, drafts, heads, kv, dim, page, dtype):
    c = Case(contexts, drafts, heads, kv, dim, page, dtype)
    lse = torch.empty(c.q.shape[:2], device="cuda")
    out = c.run(lse=lse)
    o, bound, want = c.expected()
    check(out, o, bound)
    assert (lse.double() - want).abs().max().item() <= 2.0 ** -24 * (3 * dim * 8 + 64)
    # Other splits of the same work, and a second call.
    for most in (0, 100, max(contexts), 1 << 20):
        check(c.run(max_context=most), o, bound)
    assert torch.equal(c.run(), out)


@pytest.mark.parametrize("drafts", [[1, 1, 1], [4, 1, 3]])
def test_without_masks_a_token_sees_the_drafts_up_to_itself(drafts):
    c = Case([50, 200, 33], drafts, 8, 2, 128, 16, torch.bfloat16)
    c.sees = [set(range(t + 1)) for d in drafts for t in range(d)]
    o, bound, _ = c.expected()
    check(c.run(masks=None), o, bound)
    assert torch.equal(c.run(masks=None), c.run())


@pytest.mark.parametrize("context", [0, 40])
def test_rows_whose_mask_leaves_nothing(context):
    """No drafted token, not even itself: zeros without a context, the context alone with one."""
    c = Case([context, 30], [5, 2], 4, 2, 64, 16, torch.bfloat16)
    c.sees[1] = set()
    c.sees[3] = {0}
    lse = torch.zeros(7, 4, device="cuda")
    out = c.run(lse=lse)
    o, bound, want = c.expected()
    check(out, o, bound)
    if context == 0:
        assert float(out[1].abs().max()) == 0.0 and bool((lse[1] == float("-inf")).all())
        assert torch.equal(lse == float("-inf"), want == float("-inf"))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("heads,kv", [(8, 2), (40, 8), (40, 2)])
def test_bad_values_of_an_unseen_draft(heads, kv, dtype):
    """A drafted token's NaN key or infinite value reaches its descendants alone."""
    c = Case([45, 20], [9, 4], heads, kv, 128, 16, dtype)
    clean = c.run()
    page = c.table[c.slots[0], (45 + 4) // 16].item()
    row = (45 + 4) % 16
    see = torch.tensor([4 in s and i < 9 for i, s in enumerate(c.sees)], device="cuda")
    group = heads // kv
    v = c.v.clone()
    v[page, 1, row, 3] = float("inf")
    out = c.run(v_pages=v)
    hit = torch.zeros(out.shape, dtype=torch.bool, device="cuda")
    hit[see, group:2 * group, 3] = True
    assert torch.equal(out[~hit], clean[~hit]) and bool((out[hit].float() == float("inf")).all())
    k = c.k.clone()
    k[page, 1, row] = float("nan")
    out = c.run(k_pages=k)
    hit[see, group:2 * group] = True
    assert torch.equal(out[~hit], clean[~hit]) and bool(torch.isnan(out[hit]).all())


@pytest.mark.parametrize("contexts,drafts,heads,kv", [([45, 20], [3, 4], 8, 2), ([3000, 200], [3, 4], 8, 2), ([14000], [2], 4, 4),
                                                      ([2000, 90], [30, 9], 40, 8)])
def test_a_nan_query_gives_nan_and_no_other_row_does(contexts, drafts, heads, kv):
    """However a row's keys are split: with every score NaN no part has a maximum, and the sums still tell."""
    c = Case(contexts, drafts, heads, kv, 128, 16, torch.bfloat16)
    clean = c.run()
    q = c.q.clone()
    q[1, 2, 70] = float("nan")
    lse = torch.empty(c.q.shape[:2], device="cuda")
    out = c.run(q=q, lse=lse)
    hit = torch.zeros(out.shape, dtype=torch.bool, device="cuda")
    hit[1, 2] = True
    assert bool(torch.isnan(out[hit]).all()) and torch.equal(out[~hit], clean[~hit])
    assert torch.equal(torch.isnan(lse), hit[..., 0])


def test_pages_of_another_layout_and_a_strided_table():
    """Positions outermost in a page, and a table that is part of a wider one."""
    c = Case([100, 260], [6, 2], 8, 4, 64, 32, torch.float16)
    o, bound, _ = c.expected()
    k, v = (x.transpose(1, 2).contiguous().transpose(1, 2) for x in (c.k, c.v))
    wide = torch.full((c.table.shape[0], c.table.shape[1] + 7), 1 << 30, dtype=torch.int32, device="cuda")
    wide[:, 2:2 + c.table.shape[1]] = c.table
    out = torch.full((8, 9, 64), 2.0, dtype=torch.float16, device="cuda")
    c.run(k_pages=k, v_pages=v, page_table=wide[:, 2:2 + c.table.shape[1]], out=out[:, 1:])
    check(out[:, 1:], o, bound)
    assert bool((out[:, 0] == 2.0).all())


def test_a_pool_beyond_32_bits():
    """Pages past 2^32 bytes and 2^31 elements of the pool."""
    c = Case([150], [3], 8, 8, 128, 32, torch.bfloat16)
    o, bound, _ = c.expected()
    far = 70000
    k, v = (torch.empty(far + c.n_pages, 8, 32, 128, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    assert k.numel() > 1 << 31
    k[far:], v[far:] = c.k, c.v
    check(c.run(k_pages=k, v_pages=v, page_table=torch.where(c.table >= 0, c.table + far, -1)), o, bound)


def test_slots_and_pages_that_do_not_exist():
    """Unknown slots give zeros; page numbers outside the pool read page 0, lengths past the table are bounded."""
    c = Case([40, 50], [2, 2], 4, 2, 64, 16, torch.bfloat16)
    out = c.run(seqs=_ints([c.slots[0], 99]))
    o, bound, _ = c.expected()
    check(out[:2], o[:2], bound[:2])
    assert float(out[2:].abs().max()) == 0.0
    out = c.run(seqs=_ints([c.slots[0], -1]))
    assert float(out[2:].abs().max()) == 0.0
    k, v = torch.nan_to_num(c.k), torch.nan_to_num(c.v)
    table = c.table.clone()
    table[c.slots[1], 1], table[c.slots[1], 2] = 1 << 30, -7
    lengths = c.lengths.clone()
    lengths[c.slots[1]] = 1 << 30
    assert bool(torch.isfinite(c.run(k_pages=k, v_pages=v, page_table=table, lengths=lengths)).all())


def test_masks_from_parents():
    c = Case([5, 9, 3], [70, 1, 130], 2, 1, 64, 16, torch.bfloat16)
    got = tree_masks(_ints(c.parents), c.offsets, 130)
    assert torch.equal(got, c.bits())
    # A parent that is not an earlier token starts a path.
    assert tree_masks(_ints([5, 7, 1, -3]), _ints([0, 4]), 4).tolist() == [[1], [2], [6], [8]]


def test_replayed_from_a_graph():
    c = Case([900, 130], [6, 3], 40, 8, 128, 16, torch.bfloat16)
    masks, out = c.bits(), torch.zeros_like(c.q)
    c.run(masks=masks, out=out)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        c.run(masks=masks, out=out)
    for length in (900, 200, 31, 899):
        c.lengths[c.slots[0]] = length
        graph.replay()
        torch.cuda.synchronize()
        got = out.clone()
        assert torch.equal(got, c.run(masks=masks))
        torch.cuda.synchronize()


def test_another_stream():
    c = Case([3000, 130], [6, 3], 40, 8, 128, 16, torch.bfloat16)
    first = c.run()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = [c.run() for _ in range(4)]
    side.synchronize()
    assert all(torch.equal(x, first) for x in again)


def test_nothing_to_do():
    c = Case([40], [2], 4, 2, 64, 16, torch.bfloat16)
    empty = torch.empty(0, 4, 64, dtype=torch.bfloat16, device="cuda")
    assert c.run(q=empty, seqs=_ints([]), draft_offsets=_ints([0]), masks=None).shape == (0, 4, 64)
    # A sequence without drafted tokens among others.
    d = Case([40, 20, 30], [2, 0, 1], 4, 2, 64, 16, torch.bfloat16)
    o, bound, _ = d.expected()
    check(d.run(), o, bound)


def test_refusals():
    c = Case([40], [2], 4, 2, 64, 16, torch.bfloat16)
    for bad, message in [
        (dict(q=c.q.half()), "k_pages must be"), (dict(v_pages=c.v[:2]), "k_pages' shape"), (dict(q=c.q[:, :3]), "multiple of their"),
        (dict(page_table=c.table.long()), "int32"), (dict(lengths=c.lengths[:1]), "lengths"), (dict(seqs=c.seqs.long()), "int32"),
        (dict(draft_offsets=_ints([0, 1, 2])), "one entry more"), (dict(max_drafts=0), "at least 1"),
        (dict(masks=c.bits().int()), "int64"), (dict(masks=c.bits(), max_drafts=65), "at least 2"), (dict(max_context=-1), "negative"),
        (dict(scale=0.0), "positive"), (dict(k_pages=c.k[..., 1:], v_pages=c.v[..., 1:]), "16-byte|dim"),
        (dict(out=torch.empty(1, 4, 64, dtype=torch.bfloat16, device="cuda")), "q's shape"),
    ]:
        with pytest.raises(ValueError, match=message):
            c.run(**bad)
    with pytest.raises(RuntimeError, match="GPU only"):
        c.run(k_pages=c.k.cpu(), v_pages=c.v.cpu())
