"""What the cache's steps do with numbers on the GPU that no correct program passes."""
import pytest
import torch

from tests.test_gpu_kv_cache import Pair, _ints

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("first", [-(1 << 31), -(1 << 31) + 1, -(1 << 30), -1000])
def test_append_with_offsets_far_below_zero(first):
    """The rows' positions lie past every page: nothing is written."""
    p = Pair()
    p.write([0, 3], [5, 1])
    before = p.cache.pool.clone()
    k = torch.zeros(3, p.HEADS, p.DIM, dtype=torch.bfloat16, device="cuda")
    p.cache.append(1, k, k, _ints([3]), _ints([first, 3]))
    with pytest.raises(RuntimeError, match="past a sequence's pages"):
        p.cache.check()
    assert torch.equal(p.cache.pool, before)
    p.check()


@pytest.mark.parametrize("drop", [1, 2, 9, 1 << 30])
def test_advance_does_not_shorten(drop):
    """Offsets that fall are reported, so a length cannot come to lie inside a page that another slot shares."""
    p = Pair()
    p.write([0, 3], [9, 1])
    p.fork([0], [1])
    p.cache.advance(_ints([1]), _ints([drop, 0]))
    with pytest.raises(RuntimeError, match="does not exist"):
        p.cache.check()
    p.check()
    # The branch goes on, and its source keeps its rows.
    p.write([1], [2])
    p.check()
