"""Rows beside those that a call leaves out: they are written, with their own values, and nothing else is."""
import pytest
import torch

from afterimage_amd.runtime.attention import rotary_tables
from afterimage_amd.runtime.kv_cache import PagedKVCache
from tests.eight_bits import Copy, turn

pytestmark = pytest.mark.gpu

KINDS = [torch.bfloat16, torch.float16, torch.float8_e4m3fn]
PROBLEM = {"none": None, "index": "does not exist", "full": "past a sequence's pages"}


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def make(kind, slots=3):
    cache = PagedKVCache.allocate(1, 8, 16, 2, 64, slots, 3, kind)
    cache.pool.view(torch.uint8 if kind is torch.float8_e4m3fn else torch.int16).zero_()
    if cache.scales is not None:
        cache.scales.fill_(1.0)
    return cache


def checked(cache, problem):
    if PROBLEM[problem] is None:
        cache.check()
    else:
        with pytest.raises(RuntimeError, match=PROBLEM[problem]):
            cache.check()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("half", [32, 12])
@pytest.mark.parametrize("slots,offsets,positions,turned,stored,problem", [
    ([0], [2, 6], None, range(2, 6), range(2, 6), "none"),                                       # rows of no sequence before and after
    ([0], [0, 12], None, range(8), range(8), "index"),                                           # positions 8 .. 11 have no angles
    ([0], [0, 12], [7, 8, 0, -1, 3, 99, 2, 2, 1 << 30, 5, 6, 7], [0, 2, 4, 6, 7, 9, 10, 11], [0, 2, 4, 6, 7, 9, 10, 11], "index"),
    ([0, 44, 0], [0, 3, 7, 7], None, range(3), range(3), "index"),                               # a slot that does not exist, an empty sequence
    ([1], [0, 4], None, range(4), [], "full"),                                                   # no page: the queries turn all the same
    ([0], [0, 12], [0] * 12, range(12), range(12), "none"),
])
def test_appended(kind, interleaved, half, slots, offsets, positions, turned, stored, problem):
    dtype = torch.float16 if kind is torch.float16 else torch.bfloat16
    cache = make(kind)
    cache.reserve(ints([0]), ints([16]))
    g = torch.Generator().manual_seed(half)
    q, k, v = (torch.randn(12, h, 64, generator=g).to(dtype) for h in (4, 2, 2))
    cos, sin = rotary_tables(8, 2 * half, 100.0, "cpu")
    out = torch.full_like(q, 5.0).cuda()
    copy = Copy(cache)
    cache.append_rotated(0, q.cuda(), k.cuda(), v.cuda(), ints(slots), ints(offsets), cos.cuda(), sin.cuda(),
                         None if positions is None else ints(positions), interleaved=interleaved, out=out)
    checked(cache, problem)
    at = torch.tensor(positions if positions else [max(0, r - offsets[0]) for r in range(12)]).clamp(0, 7)
    tq, tk = (turn(x.float(), cos[at], sin[at], interleaved) for x in (q, k))
    want = torch.full_like(q, 5.0)
    want[list(turned)] = tq[list(turned)].to(dtype)
    assert torch.equal(out.cpu(), want)
    if len(stored):
        page = int(copy.table[0, 0])
        rows = [r - offsets[0] for r in stored]
        for which, x in ((0, tk), (1, v.float())):
            for head in range(2):
                part = x[list(stored), head].double()
                if copy.wide:
                    copy.pool[0, which, page, head, rows] = part.to(kind)
                else:
                    # The block is formed from the rows that are stored; the others' places stay.
                    scale = 2.0 ** -100
                    while float(part.abs().max()) > 448.0 * scale:
                        scale *= 2.0
                    copy.pool[0, which, page, head, rows] = (part / scale).float().to(kind).double()
                    copy.scales[0, which, page, head, 0] = scale
    copy.same(cache)


@pytest.mark.parametrize("kind", KINDS)
def test_read(kind):
    """The second row of a sequence lies past its pages; a slot that does not exist, one without pages; rows of no sequence."""
    cache = make(kind, slots=4)
    cache.reserve(ints([0, 2]), ints([16, 33]))
    g = torch.Generator(device="cuda").manual_seed(3)
    x = (torch.randn(cache.pool.shape, generator=g, device="cuda") * 40).clamp(-400, 400)
    cache.pool.copy_(x.to(kind))
    copy = Copy(cache)
    dtype = torch.bfloat16 if kind is torch.float8_e4m3fn else kind
    out = tuple(torch.full((9, 2, 64), 7.0, dtype=dtype, device="cuda") for _ in range(2))
    cache.read(0, ints([2, 9, 1, 0]), ints([1, 3, 5, 6, 8]), 9, ints([47, 0, 0, 14]), out=out)
    with pytest.raises(RuntimeError, match="past a sequence's pages.*does not exist"):
        cache.check()
    for which in range(2):
        want = torch.full((9, 2, 64), 7.0, dtype=torch.float64)
        for row, slot, position in ((1, 2, 47), (6, 0, 14), (7, 0, 15)):
            want[row] = torch.stack([copy.row(0, which, head, slot, position).double() for head in range(2)])
        assert torch.equal(out[which].cpu().double(), want.to(dtype).double())
