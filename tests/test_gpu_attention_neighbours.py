"""A row's result is bit for bit its own: keys that only its neighbours in a
wave see do not change its last bits, however large their scores."""
import pytest
import torch

from afterimage_amd.runtime.attention import prompt_attention
from tests.test_gpu_prompt_attention import _case, _offsets
from tests.test_gpu_tree_attention import Case

pytestmark = pytest.mark.gpu

# Scores of tens to hundreds of octaves: the number that probabilities are taken against is raised again and again.
SCALE = 1.0


@pytest.mark.parametrize("factor", [40.0, float("inf"), float("nan")])
@pytest.mark.parametrize("rows,keys,heads,kv,dim", [([300], [300], 2, 1, 64), ([90, 40], [400, 40], 4, 2, 128), ([20], [3000], 4, 1, 64),
                                                    ([70], [70], 2, 1, 256)])
def test_prompts(rows, keys, heads, kv, dim, factor):
    q, k, v = _case(rows, keys, heads, kv, dim, torch.bfloat16)
    clean = prompt_attention(q, k, v, _offsets(rows), _offsets(keys), scale=SCALE)
    for back in (1, 7, rows[0] // 2, rows[0] - 1):
        k2 = k.clone()
        at = keys[0] - back  # the last `back` rows of the first sequence see it
        k2[at] = k2[at] * factor
        out = prompt_attention(q, k2, v, _offsets(rows), _offsets(keys), scale=SCALE)
        blind = torch.ones(sum(rows), dtype=torch.bool, device="cuda")
        blind[rows[0] - back:rows[0]] = False
        assert torch.equal(out[blind], clean[blind]), back


@pytest.mark.parametrize("factor", [40.0, float("inf"), float("nan")])
@pytest.mark.parametrize("contexts,drafts,heads,kv,page", [([45, 20], [9, 4], 4, 2, 16), ([900], [12], 40, 8, 64), ([70, 2000], [64, 40], 8, 2, 16)])
def test_trees(contexts, drafts, heads, kv, page, factor):
    c = Case(contexts, drafts, heads, kv, 128, page, torch.float16)
    clean = c.run(scale=SCALE)
    for drafted in (0, 2, drafts[0] // 2, drafts[0] - 1):
        k = c.k.clone()
        at = contexts[0] + drafted
        row = k[c.table[c.slots[0], at // page], :, at % page]
        row.mul_(factor)
        blind = torch.tensor([i >= drafts[0] or drafted not in s for i, s in enumerate(c.sees)], device="cuda")
        out = c.run(k_pages=k, scale=SCALE)
        assert torch.equal(out[blind], clean[blind]), drafted
