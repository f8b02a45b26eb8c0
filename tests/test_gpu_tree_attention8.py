"""Attention over a cache in 8 bits against its definition in 64 bits.

The elements are what the codes and scales stand for, and enter the first
product exactly, so the bounds are those of attention over 16 bits
(attention_oracle), with probabilities rounded to bf16 whatever the queries'
type: 2^-8 A in place of the type's own, and in fp16 no term for probabilities
that are not normal there (bf16 has fp32's range). Multiplying a score by its
key's scale is exact: scales are powers of two.
"""
import pytest
import torch

from afterimage_amd.runtime.attention import tree_attention, tree_masks
from tests.attention_oracle import UNIT, check

pytestmark = pytest.mark.gpu


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def attend(q, k, v, visible, scale):
    """(o, bound, lse) in 64 bits; k and v in 64 bits already."""
    n, heads, dim = q.shape
    m, kv = k.shape[:2]
    u, x = UNIT[q.dtype], q.double()
    k, v = (t.repeat_interleave(heads // kv, 1) for t in (k, v))
    s = torch.matmul(x.transpose(0, 1), k.permute(1, 2, 0).contiguous()) * scale
    size = (torch.matmul(x.abs().transpose(0, 1), k.abs().permute(1, 2, 0).contiguous()) * scale).masked_fill(~visible, 0.0)
    s = s.masked_fill(~visible, float("-inf"))
    lse = torch.logsumexp(s, -1)
    p = torch.exp(s - lse.masked_fill(lse == float("-inf"), 0.0)[..., None])
    vt = v.transpose(0, 1).contiguous()
    o, a = torch.matmul(p, vt).transpose(0, 1), torch.matmul(p, vt.abs()).transpose(0, 1)
    most = size.amax(-1).clamp_min(1.0).t()[..., None]
    bound = (2.0 ** -8 + 2.0 ** -24 * (2 * (dim + 8) * most + 2 * m)) * a + u * o.abs()
    if q.dtype == torch.float16:
        bound = bound + 2.0 ** -25
    return o, bound, lse.t()


class Case:
    """Sequences in a pool whose other pages, and rows past the drafted ones, are NaN."""

    def __init__(self, lengths, drafts, heads, kv, dim, page, dtype, seed=0, spread=4, layers=1):
        g = torch.Generator().manual_seed(seed)
        self.lengths, self.drafts, self.dtype = lengths, drafts, dtype
        count = [-(-(a + b) // page) for a, b in zip(lengths, drafts)]
        n_pages = sum(count) + 2
        order = torch.randperm(n_pages, generator=g).tolist()
        self.table, at = [], 0
        for c in count:
            self.table.append(order[at:at + c])
            at += c
        shape = (2, n_pages, kv, page, dim)
        codes = (torch.randn(shape, generator=g) * 100).clamp(-448, 448).to(torch.float8_e4m3fn)
        scales = torch.exp2(torch.randint(-spread, spread // 2 + 1, (2, n_pages, kv, page // 16), generator=g).float() - 6)
        raw = codes.view(torch.uint8)
        used = torch.zeros(n_pages, page, dtype=torch.bool)
        for row, a, b in zip(self.table, lengths, drafts):
            for j in range(a + b):
                used[row[j // page], j % page] = True
        raw.masked_fill_(~used[None, :, None, :, None], 0x7F)
        scales.masked_fill_(~used.view(n_pages, -1, 16).any(-1)[None, :, None], float("nan"))
        self.codes, self.scales = codes.cuda(), scales.cuda()
        self.q = (torch.randn(sum(drafts), heads, dim, generator=g) * 0.5).to(dtype).cuda()
        most = max(map(len, self.table))
        self.page_table = ints([r + [-1] * (most - len(r)) for r in self.table])
        self.offsets = ints([sum(drafts[:i]) for i in range(len(drafts) + 1)])
        self.page = page

    def run(self, masks=None, **options):
        n = len(self.lengths)
        return tree_attention(self.q, self.codes[0], self.codes[1], self.page_table, ints(self.lengths), ints(list(range(n))), self.offsets, masks,
                              max_drafts=max(self.drafts), k_scales=self.scales[0], v_scales=self.scales[1], **options)

    def rows(self, which, b):
        """Sequence b's keys or values [positions, kv, dim] in 64 bits."""
        x = self.codes[which].cpu().double() * self.scales[which].cpu().double().repeat_interleave(16, -1)[..., None]
        j = torch.arange(self.lengths[b] + self.drafts[b])
        return x[torch.tensor(self.table[b])[j // self.page], :, j % self.page].cuda()

    def compare(self, got, seen=None, scale=None, lse=None):
        scale = scale or self.q.shape[2] ** -0.5
        at = 0
        for b, (a, n) in enumerate(zip(self.lengths, self.drafts)):
            j, t = torch.arange(a + n, device="cuda"), torch.arange(n, device="cuda")[:, None]
            visible = j <= a + t if seen is None else (j < a) | seen[at:at + n, (j - a).clamp_min(0)]
            o, bound, log = attend(self.q[at:at + n], self.rows(0, b), self.rows(1, b), visible, scale)
            check(got[at:at + n], o, bound, "sequence %d" % b)
            if lse is not None:
                # The sum's relative error and the exponentials' arguments', as in the bound; 2^-20 of the logarithm itself.
                size = (self.q[at:at + n].double().abs().amax(-1) * self.rows(0, b).abs().amax((0, 2)).repeat_interleave(self.q.shape[1] // self.codes.shape[2])
                        * self.q.shape[2] * scale)
                assert bool(((lse[at:at + n] - log).abs() <= 2.0 ** -24 * (2 * (self.q.shape[2] + 8) * size.clamp_min(1.0) + 2 * (a + n)) + 2.0 ** -20 * log.abs()).all())
            at += n
        return got


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("heads,kv,dim", [(5, 1, 128), (4, 2, 64), (8, 8, 16), (6, 2, 96), (4, 1, 256), (3, 3, 208), (32, 4, 48)])
@pytest.mark.parametrize("page", [16, 48, 64])
def test_single_tokens(dtype, heads, kv, dim, page):
    case = Case([0, 1, 15, 16, 31, 64, 200, 517], [1] * 8, heads, kv, dim, page, dtype, seed=dim + page)
    lse = torch.zeros(8, heads, device="cuda")
    case.compare(case.run(lse=lse), lse=lse)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("heads,kv,dim,drafts", [(5, 1, 128, [9, 1, 12]), (40, 8, 128, [33, 1, 7]), (8, 2, 64, [16, 40, 3]), (4, 2, 256, [20, 2, 30]),
                                                 (16, 1, 96, [8, 5, 3]), (2, 1, 32, [70, 64, 65])])
@pytest.mark.parametrize("page", [16, 32])
def test_drafted_trees(dtype, heads, kv, dim, drafts, page):
    case = Case([37, 700, 0], drafts, heads, kv, dim, page, dtype, seed=dim)
    parents, g = [], torch.Generator().manual_seed(1)
    for n in drafts:
        parents += [-1] + [int(torch.randint(max(0, t - 5), t, (1,), generator=g)) for t in range(1, n)]
    masks = tree_masks(ints(parents), case.offsets, max(drafts))
    bits = masks.cpu()
    seen = torch.zeros(sum(drafts), max(drafts), dtype=torch.bool)
    for j in range(max(drafts)):
        seen[:, j] = (bits[:, j // 64] >> (j % 64)) & 1 == 1
    case.compare(case.run(masks), seen.cuda())
    case.compare(case.run())


@pytest.mark.parametrize("heads,kv,drafts", [(5, 1, [1, 1]), (8, 1, [6, 8]), (40, 8, [4, 30])])
def test_long_contexts_are_split_and_joined(heads, kv, drafts):
    case = Case([9000, 4100], drafts, heads, kv, 128, 32, torch.bfloat16, seed=3)
    got = case.compare(case.run(max_context=9000))
    assert torch.equal(got, case.run(max_context=9000))
    # Parts may be cut anywhere: what a call expects changes how, and the result by roundings.
    case.compare(case.run(max_context=100))
    case.compare(case.run())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_scales_far_apart(dtype):
    """Scales from 2^-40 to 2^20 side by side: values past fp16's range inside the sums, for queries in fp16 too."""
    case = Case([90], [2], 2, 1, 64, 16, dtype, seed=5)
    block = torch.arange(case.scales[0].numel(), device="cuda").view(case.scales[0].shape)
    fine = ~case.scales.isnan()
    case.scales[0] = torch.where(fine[0], torch.exp2(((block * 5) % 12).float() - 16), case.scales[0])
    case.scales[1] = torch.where(fine[1], torch.exp2(((block * 7) % 20).float() - 22), case.scales[1])
    case.compare(case.run())


@pytest.mark.parametrize("heads,drafts", [(2, 3), (5, 30), (8, 8)])
def test_what_a_row_does_not_see_does_not_reach_it(heads, drafts):
    """NaN in drafted keys and values that a row's mask leaves out; the rows that see them are NaN."""
    case = Case([50], [drafts], heads, 1, 64, 16, torch.bfloat16, seed=7)
    masks = tree_masks(ints([-1] * drafts), case.offsets, drafts)  # every token sees the context and itself
    clean = case.run(masks)
    for which in (0, 1):
        codes = case.codes.clone()
        at = 50 + drafts - 1
        case.codes.view(torch.uint8)[which, case.table[0][at // 16], :, at % 16, 3::2] = 0x7F
        got = case.run(masks)
        assert torch.equal(got[:-1], clean[:-1])
        assert bool(got[-1].isnan().any())
        case.codes.copy_(codes)


def test_rows_that_see_nothing():
    case = Case([0, 3], [2, 2], 4, 2, 64, 16, torch.bfloat16)
    lse = torch.zeros(4, 4, device="cuda")
    got = case.run(torch.zeros(4, 1, dtype=torch.int64, device="cuda"), lse=lse)
    assert bool((got[:2] == 0).all()) and bool((lse[:2] == float("-inf")).all()) and bool((got[2:] != 0).any())


def test_pages_and_slots_that_do_not_exist():
    """Bad page numbers read page 0, an unknown slot gives zeros, rows of no sequence stay; nothing leaves the pool."""
    case = Case([40, 20], [2, 2], 4, 2, 64, 16, torch.bfloat16)
    case.codes.view(torch.uint8).copy_(torch.where(case.codes.isnan(), torch.zeros((), dtype=torch.uint8, device="cuda"), case.codes.view(torch.uint8)))
    case.scales.nan_to_num_(1.0)
    case.page_table[0, 1] = 1 << 30
    case.page_table[0, 2] = -5
    out = torch.full_like(case.q, 3.0)
    got = tree_attention(case.q, case.codes[0], case.codes[1], case.page_table, ints([40, 20]), ints([0, 9]), ints([0, 2, 3]), max_drafts=2,
                         k_scales=case.scales[0], v_scales=case.scales[1], out=out)
    assert bool(torch.isfinite(got[:2]).all()) and bool((got[2] == 0).all()) and bool((got[3] == 3.0).all())


def test_pages_of_one_pool_for_all_layers():
    """Keys, values and scales as strided views of larger tensors, heads last but one."""
    case = Case([77, 130], [3, 1], 8, 4, 64, 32, torch.bfloat16, seed=9)
    want = case.run()
    n_pages, kv, page, dim = case.codes.shape[1:]
    turned = torch.zeros(2, n_pages, page, 2 * kv, dim, dtype=torch.uint8, device="cuda")
    turned[..., kv:, :] = case.codes.view(torch.uint8).transpose(2, 3)
    views = turned.view(torch.float8_e4m3fn)[..., kv:, :].transpose(2, 3)
    wide = torch.zeros(2, kv, n_pages, 2 * (page // 16), device="cuda")
    wide[..., :page // 16] = case.scales.transpose(1, 2)
    scales = wide[..., :page // 16].transpose(1, 2)
    got = tree_attention(case.q, views[0], views[1], case.page_table, ints(case.lengths), ints([0, 1]), case.offsets, max_drafts=3,
                         k_scales=scales[0], v_scales=scales[1])
    assert torch.equal(got, want)
