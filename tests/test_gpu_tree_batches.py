"""Many trees a call, and many drafted tokens without masks."""
import random

import pytest
import torch

from tests.attention_oracle import check
from tests.test_gpu_tree_attention import Case

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("long", [0, 70, 139])
def test_more_sequences_than_a_wave_has_lanes(long):
    """140 of them, empty ones among them; one is long enough for many parts, which the join looks for."""
    rng = random.Random(long)
    contexts = [rng.randint(0, 60) for _ in range(140)]
    contexts[long] = 17000
    drafts = [rng.choice((0, 1, 1, 2, 3)) for _ in range(140)]
    drafts[long] = 2
    c = Case(contexts, drafts, 4, 2, 64, 16, torch.bfloat16, seed=long)
    o, bound, _ = c.expected()
    for longest in (17000, 60, 1 << 20):
        check(c.run(max_context=longest), o, bound)


@pytest.mark.parametrize("drafts,context,heads,kv", [([300], 0, 4, 2), ([130, 257], 100, 4, 2), ([600, 3, 64], 700, 8, 1)])
def test_many_drafted_rows_without_masks(drafts, context, heads, kv):
    """A stretch of a prompt over the cache: a row sees the context and the rows up to its own."""
    c = Case([context] * len(drafts), drafts, heads, kv, 64, 16, torch.bfloat16)
    c.sees = [set(range(t + 1)) for d in drafts for t in range(d)]
    o, bound, _ = c.expected()
    check(c.run(masks=None), o, bound)
    assert torch.equal(c.run(masks=None), c.run())
