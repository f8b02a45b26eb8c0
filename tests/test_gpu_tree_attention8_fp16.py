"""fp16 queries over a cache in 8 bits: probabilities keep 16 bits.

A probability is the sum of two bf16 numbers: the nearest, which is off by 2^-8
of it at most, and the nearest to what is left, off by 2^-8 of that. So the
bound of attention_oracle holds with 2^-16 A in place of the type's own u A, no
term for probabilities that are not normal in fp16, and n terms more in the
result's sum, each of which is two products. Contexts are short and heads narrow
enough that probabilities of one bf16 number would not pass (which a test on the
CPU shows of the same inputs).
"""
import pytest
import torch

from afterimage_amd.runtime.attention import tree_attention
from tests.attention_oracle import check

CASES = [  # lengths, drafts, heads, kv_heads, dim, page
    ([2, 5, 9, 15, 16, 31], [1] * 6, 4, 2, 64, 16),
    ([3, 7, 30], [1, 1, 1], 5, 1, 128, 48),
    ([4, 13, 40], [1, 1, 1], 8, 8, 16, 64),
    ([6, 21], [1, 1], 6, 2, 96, 16),
    ([8, 20], [1, 1], 4, 1, 256, 16),
    ([11, 3], [9, 12], 5, 1, 128, 16),      # 64 rows of a head's group
    ([17, 5], [30, 33], 40, 8, 64, 32),     # more, tiles shared
    ([12, 2], [20, 30], 8, 2, 256, 64),
]


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


class Inputs:
    """Queries, pages that lie in a sequence's order, their scales; keys and values of a sequence in 64 bits."""

    def __init__(self, lengths, drafts, heads, kv, dim, page):
        g = torch.Generator().manual_seed(1000 * dim + len(lengths))
        self.lengths, self.drafts, self.page = lengths, drafts, page
        count = [-(-(a + n) // page) for a, n in zip(lengths, drafts)]
        self.table = [list(range(sum(count[:b]), sum(count[:b + 1]))) for b in range(len(count))]
        shape = (2, sum(count), kv, page, dim)
        self.codes = (torch.randn(shape, generator=g) * 100).clamp(-448, 448).to(torch.float8_e4m3fn)
        self.scales = torch.exp2(torch.randint(-2, 2, (*shape[:3], page // 16), generator=g).float() - 7)
        self.q = (torch.randn(sum(drafts), heads, dim, generator=g) * 0.5).half()

    def rows(self, which, b):
        x = self.codes[which].double() * self.scales[which].double().repeat_interleave(16, -1)[..., None]
        j = torch.arange(self.lengths[b] + self.drafts[b])
        return x[torch.tensor(self.table[b])[j // self.page], :, j % self.page]

    def sequences(self):
        """(rows of q, o, bound, probabilities, values) of each sequence in 64 bits; probabilities of largest 1."""
        at = 0
        for b, (a, n) in enumerate(zip(self.lengths, self.drafts)):
            q = self.q[at:at + n].double()
            heads, dim = q.shape[1:]
            k, v = (self.rows(which, b) for which in range(2))
            group = heads // k.shape[1]
            k, v = (x.repeat_interleave(group, 1).transpose(0, 1).contiguous() for x in (k, v))
            m, q = a + n, q.transpose(0, 1)
            unseen = torch.arange(m) > a + torch.arange(n)[:, None]
            s = torch.matmul(q, k.transpose(1, 2).contiguous()) * dim ** -0.5
            most = (torch.matmul(q.abs(), k.abs().transpose(1, 2).contiguous()) * dim ** -0.5).masked_fill(unseen, 0.0).amax(-1).clamp_min(1.0)
            s = s.masked_fill(unseen, float("-inf"))
            p = torch.exp(s - s.amax(-1, keepdim=True))
            total = p.sum(-1, keepdim=True)
            o, size = torch.matmul(p, v) / total, torch.matmul(p, v.abs()) / total
            bound = (2.0 ** -16 + 2.0 ** -24 * (2 * (dim + 8) * most[..., None] + 3 * m)) * size + 2.0 ** -11 * o.abs() + 2.0 ** -25
            yield slice(at, at + n), o.transpose(0, 1), bound.transpose(0, 1), p, v
            at += n


@pytest.mark.gpu
@pytest.mark.parametrize("case", CASES)
def test_probabilities_keep_sixteen_bits(case):
    x = Inputs(*case)
    most = max(map(len, x.table))
    codes, scales = x.codes.cuda(), x.scales.cuda()
    offsets = ints([sum(x.drafts[:b]) for b in range(len(x.drafts) + 1)])
    got = tree_attention(x.q.cuda(), codes[0], codes[1], ints([row + [-1] * (most - len(row)) for row in x.table]), ints(x.lengths),
                         ints(list(range(len(x.lengths)))), offsets, max_drafts=max(x.drafts), k_scales=scales[0], v_scales=scales[1]).cpu()
    for at, o, bound, _, _ in x.sequences():
        check(got[at], o, bound, "rows %s" % at)


@pytest.mark.parametrize("case", CASES)
def test_the_bound_tells_one_bf16_number_from_two(case):
    """The definition with probabilities of two bf16 numbers, rounded to fp16, lies within it, in every sequence; of one, in none."""
    for at, o, bound, p, v in Inputs(*case).sequences():
        first = p.bfloat16().double()
        for kept, passes in ((first, False), (first + (p - first).bfloat16().double(), True)):
            got = (torch.matmul(kept, v) / p.sum(-1, keepdim=True)).transpose(0, 1).half().double()
            assert bool(((got - o).abs() <= 1.05 * bound).all()) == passes, "rows %s" % at
