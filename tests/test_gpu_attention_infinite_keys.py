"""A key whose score is -inf weighs nothing, wherever in its row the infinite element is."""
import pytest
import torch

from afterimage_amd.runtime.attention import prompt_attention
from tests.attention_oracle import attend, check
from tests.test_gpu_prompt_attention import _case, _offsets
from tests.test_gpu_tree_attention import Case

pytestmark = pytest.mark.gpu


def _minus_infinity(q, k, keys, column):
    """Element `column` of these keys is -inf, and that of every query positive."""
    q[..., column] = q[..., column].abs() + 0.25
    for j in keys:
        k[j, :, column] = float("-inf")


@pytest.mark.parametrize("dim", [8, 40, 64, 72, 96, 128, 168, 248, 256])
@pytest.mark.parametrize("rows,keys", [([200], [330]), ([9, 70], [2900, 100])])
@pytest.mark.parametrize("column", [-1, -8, 0])
def test_prompts(rows, keys, dim, column):
    q, k, v = _case(rows, keys, 4, 2, dim, torch.bfloat16)
    # In tiles that every row sees, on the causal edge, and in a later sequence.
    bad = [3, 70, keys[0] - rows[0] + 2] + ([sum(keys) - 1] if len(keys) > 1 else [])
    _minus_infinity(q, k, bad, column)
    out = prompt_attention(q, k, v, _offsets(rows), _offsets(keys))
    a = b = 0
    for n, m in zip(rows, keys):
        i, j = torch.arange(n, device="cuda"), torch.arange(m, device="cuda")
        visible = j <= i[:, None] + (m - n)
        for x in bad:
            if b <= x < b + m:
                visible[:, x - b] = False
        o, bound, _ = attend(q[a:a + n], torch.where(torch.isinf(k[b:b + m]), 0.0, k[b:b + m]).to(k.dtype), v[b:b + m], visible, dim ** -0.5)
        check(out[a:a + n], o, bound)
        a, b = a + n, b + m


@pytest.mark.parametrize("dim", [8, 40, 64, 72, 96, 128, 168, 248, 256])
@pytest.mark.parametrize("contexts,drafts,page", [([150, 40], [3, 2], 16), ([150, 700], [33, 9], 64), ([90, 33], [2, 40], 5)])
def test_trees(contexts, drafts, page, dim):
    c = Case(contexts, drafts, 8, 2, dim, page, torch.float16)
    parts = []
    first = 0
    c.q[..., -1] = c.q[..., -1].abs() + 0.25
    for b, (n, d) in enumerate(zip(contexts, drafts)):
        k, v = c.rows[b]
        # In a whole tile, among the last keys of the context, and a drafted token (its own row sees it too).
        bad = [1, n - 1, n + d - 1]
        for j in bad:
            c.k[c.table[c.slots[b], j // page], :, j % page, -1] = float("-inf")
        visible = torch.zeros(d, n + d, dtype=torch.bool)
        visible[:, :n] = True
        for t in range(d):
            for j in c.sees[first + t]:
                visible[t, n + j] = True
        visible[:, bad] = False
        parts.append(attend(c.q[first:first + d], k, v, visible.cuda(), dim ** -0.5))
        first += d
    o, bound, _ = (torch.cat(x) for x in zip(*parts))
    check(c.run(), o, bound)
