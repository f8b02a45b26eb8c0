"""Captured forks, releases and compactions, replayed beside the program's own calls."""
import pytest
import torch

from tests.test_gpu_kv_cache import Pair, _ints

pytestmark = pytest.mark.gpu


def _captured(step):
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    return graph


def test_a_captured_fork_beside_larger_ones():
    """Its scratch stays its own: a larger fork, and tensors made afterwards, neither disturb it nor are disturbed."""
    p = Pair(n_pages=60, max_seqs=9)
    p.write([0, 3], [10, 6])
    src, dst = _ints([0, 3]), _ints([1, 2])
    p.fork([0, 3], [1, 2])  # what a program does once before it captures
    torch.cuda.synchronize()
    graph = _captured(lambda: p.cache.fork(src, dst))
    nbytes = 4 * 2 * (2 + p.model.max_pages)
    for turn in range(4):
        p.fork([0, 0, 3, 0, 3], [4, 5, 6, 7, 8])
        p.check()
        # Tensors of the captured call's scratch's size, as the allocator would give its memory out again.
        others = [torch.full((nbytes,), 100 + i, dtype=torch.uint8, device="cuda") for i in range(8)]
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        p.model.fork([0, 3], [1, 2])
        p.check()
        assert all(bool((x == 100 + i).all()) for i, x in enumerate(others))
        p.write([0, 1, 2], [1, turn, 2])
        p.check()


def test_captured_release_and_compaction():
    p = Pair(n_pages=60)
    p.write([0, 1, 2, 3], [10, 7, 13, 9])
    slots, used = _ints([1, 4]), torch.zeros((), dtype=torch.int32, device="cuda")
    src, dst = _ints([0]), _ints([1])

    def step():
        p.cache.release(slots)
        used.copy_(p.cache.compact())
        p.cache.fork(src, dst)

    graph = _captured(step)
    for turn in range(4):
        graph.replay()
        torch.cuda.synchronize()
        p.model.release([1, 4])
        assert int(used) == p.model.compact()
        p.model.fork([0], [1])
        p.check()
        p.write([1, 4], [3, 5 + turn])
        p.fork([2], [5])
        p.release([3] if turn else [])
        p.check()


def test_forks_of_growing_size_on_another_stream():
    """A larger fork on a second stream, then memory from the first stream's pool while it may still run."""
    p = Pair(n_pages=60, max_seqs=9)
    p.write([0, 3], [10, 6])
    p.fork([0], [1])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        p.cache.fork(_ints([3]), _ints([2]))
        p.cache.fork(_ints([0, 0, 3, 0]), _ints([4, 5, 6, 7]))
    others = [torch.full((4 * (2 + p.model.max_pages),), 90 + i, dtype=torch.uint8, device="cuda") for i in range(8)]
    side.synchronize()
    torch.cuda.synchronize()
    p.model.fork([3], [2])
    p.model.fork([0, 0, 3, 0], [4, 5, 6, 7])
    p.check()
    assert all(bool((x == 90 + i).all()) for i, x in enumerate(others))
