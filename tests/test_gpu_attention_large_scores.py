"""Scores far apart and large: maxima that rise tile after tile, and parts and
waves whose maxima differ by hundreds of octaves, in every form that joins them."""
import pytest
import torch

from afterimage_amd.runtime.attention import prompt_attention
from tests.attention_oracle import check
from tests.test_gpu_prompt_attention import _case, _expected, _offsets
from tests.test_gpu_tree_attention import Case

pytestmark = pytest.mark.gpu


def _factors(m, order):
    """What each of m keys is multiplied by."""
    x = torch.linspace(0.01, 30.0, m, device="cuda")
    if order == "falling":
        x = x.flip(0)
    elif order == "stretches":  # of 200 keys, small and large in turn
        x = torch.where(torch.arange(m, device="cuda") // 200 % 2 == 0, 0.02, 20.0)
    return x[:, None, None]


@pytest.mark.parametrize("order", ["rising", "falling", "stretches"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows,keys,heads,kv,dim", [
    ([300], [300], 2, 1, 64),
    ([13], [2900], 8, 1, 128),
    ([30, 7, 2], [3000, 700, 5000], 10, 2, 64),
    ([40, 9], [1400, 2600], 8, 4, 256),
    ([5], [40000], 4, 1, 96),
])
def test_prompts(rows, keys, heads, kv, dim, dtype, order):
    q, k, v = _case(rows, keys, heads, kv, dim, dtype)
    k = torch.cat([x.float() * _factors(len(x), order) for x in k.split(keys)]).to(dtype)
    out = prompt_attention(q, k, v, _offsets(rows), _offsets(keys), scale=0.5)
    o, bound, _ = _expected(q, k, v, rows, keys, 0.5)
    check(out, o, bound)


@pytest.mark.parametrize("order", ["rising", "falling", "stretches"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("contexts,drafts,heads,kv,dim,page", [
    ([500, 7, 3000], [3, 6, 1], 40, 8, 128, 16),        # waves that deal out the keys, one tile of rows
    ([900, 2000], [12, 9], 40, 8, 128, 64),             # two tiles of rows
    ([2600, 700], [40, 33], 16, 2, 64, 64),             # shared tiles
    ([14000], [2], 4, 4, 128, 16),                      # more than 16 parts
    ([3000, 9000], [64, 5], 8, 1, 64, 5),
    ([700, 1500], [40, 9], 8, 4, 256, 32),
])
def test_trees(contexts, drafts, heads, kv, dim, page, dtype, order):
    c = Case(contexts, drafts, heads, kv, dim, page, dtype)
    for b, (k, v) in enumerate(c.rows):
        k = (k.float() * _factors(len(k), order)).to(dtype)
        c.rows[b] = (k, v)
        at = torch.arange(len(k), device="cuda")
        c.k[c.table[c.slots[b]][at // page].long(), :, at % page] = k
    o, bound, want = c.expected(0.5)
    lse = torch.empty(c.q.shape[:2], device="cuda")
    check(c.run(scale=0.5, lse=lse), o, bound)
    # The scores' own error, as in the bound, of scores of up to some thousands.
    most = max(float((c.q.float().abs().amax() * k.float().abs().amax() * dim * 0.5).item()) for k, _ in c.rows)
    assert (lse.double() - want).abs().max().item() <= 2.0 ** -24 * (2 * (dim + 8) * most + 64)
    for longest in (0, 1 << 20):
        check(c.run(scale=0.5, max_context=longest), o, bound)
