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


@pytest.mark.parametrize("count", [-1, -(1 << 31), 3, (1 << 31) - 1])
@pytest.mark.parametrize("apart", [False, True])
def test_commit_with_a_count_out_of_range(count, apart):
    """No more than accepted's width, no less than 0: the sequence stays as it is, the others are committed."""
    p = Pair()
    p.write([0, 1], [6, 3])
    p.cache.reserve(_ints([0, 1]), _ints([4, 4]))
    p.model.reserve([0, 1], [4, 4])
    numbers, _ = p.append([0, 1], [4, 4])
    new = torch.full((7,), -9, dtype=torch.int32, device="cuda") if apart else None
    p.cache.commit(_ints([0, 1]), _ints([[1, 3], [0, 2]]), _ints([count, 2]), new)
    if apart:
        assert new.tolist() == [6, 5, -9, -9, -9, -9, -9]
        p.cache.lengths[:2] = new[:2]
    p.model.rows[1] += [numbers[1][0], numbers[1][2]]
    with pytest.raises(RuntimeError, match="does not exist"):
        p.cache.check()
    p.check()
    # The drafted rows lie where they were appended.
    p.cache.commit(_ints([0]), _ints([[0, 1, 2, 3]]), _ints([4]))
    p.model.rows[0] += numbers[0]
    p.check()


@pytest.mark.parametrize("number", [-1, 40, 1 << 30])
@pytest.mark.parametrize("entry", [0, 2])
def test_forks_of_rows_with_a_page_that_does_not_exist_are_reported(number, entry):
    """A full page's entry, and the last one's."""
    p = Pair()
    p.write([0], [10])
    p.cache.page_table[0, entry] = number
    p.cache.fork(_ints([0]), _ints([1]))
    with pytest.raises(RuntimeError, match="does not exist"):
        p.cache.check()
    assert p.cache.page_table[0, entry] == number and int(p.cache.refs.sum()) <= 6


@pytest.mark.parametrize("entry", [1, 2])
def test_commits_with_a_page_that_does_not_exist_are_reported(entry):
    """Where accepted rows would go to (position 7, page 1), and where they are (8 and 10, page 2): they stay."""
    p = Pair()
    p.write([0], [7])
    p.cache.reserve(_ints([0]), _ints([5]))
    before = p.cache.pool.clone()
    p.cache.page_table[0, entry] = -5
    p.cache.commit(_ints([0]), _ints([[1]]), _ints([1]))
    with pytest.raises(RuntimeError, match="does not exist"):
        p.cache.check()
    assert torch.equal(p.cache.pool, before)
