"""Whose memory the scratch of a call is while a launch may use it. No GPU is
used: allocations and launches are recorded in place of being made there."""
import types
import weakref

import pytest
import torch

from afterimage_amd import _native
from afterimage_amd.runtime import attention, kv_cache


class Recorder:
    """torch.empty on the CPU, remembered weakly; what each launch is given."""

    def __init__(self, monkeypatch, module):
        self.made, self.launches, empty = [], [], torch.empty

        def remembered(*args, **options):
            x = empty(*args, **{**options, "device": "cpu"})
            self.made.append((x.data_ptr(), x.numel(), weakref.ref(x)))
            return x

        def launch(entry, index, *args):
            self.launches.append((args, [ref() for _, _, ref in self.made]))

        monkeypatch.setattr(torch, "empty", remembered)
        monkeypatch.setattr(module, "launch", launch)

    def living(self, address):
        """The tensor at an address of the last launch that was alive then."""
        return next((x for x in self.launches[-1][1] if x is not None and x.data_ptr() == address), None)


def _ints(*values):
    return torch.tensor(values, dtype=torch.int32)


@pytest.fixture
def cache():
    c = object.__new__(kv_cache.PagedKVCache)
    c.max_pages, c.device, c._index, c._cache = 9, torch.device("cpu"), -1, None
    c._lib = types.SimpleNamespace(aimg_cache_fork=None)
    return c


def test_a_larger_fork_takes_nothing_from_one_captured_before(cache, monkeypatch):
    """A graph that holds a fork of two pairs keeps using the scratch it was captured with."""
    seen = Recorder(monkeypatch, kv_cache)
    cache.fork(_ints(0, 0), _ints(1, 2))
    work, nbytes = seen.launches[-1][0][-2:]
    first = seen.living(work)
    assert first is not None and first.numel() >= nbytes == 4 * 2 * (2 + 9)
    kept = any(x is first for x in vars(cache).values())
    first = weakref.ref(first)
    seen.launches.clear()
    cache.fork(_ints(0, 0, 0, 0, 0), _ints(1, 2, 3, 4, 5))
    # The cache never held it (then torch's allocator decides, which knows of captures and streams), or holds it still.
    assert not kept or first() is not None


@pytest.fixture
def on_cpu(monkeypatch):
    """CPU tensors pass the attention calls' checks; their launches are recorded."""
    monkeypatch.setattr(attention, "_query", lambda q: (attention._heads(q, "q", q.dtype, -1), -1, _native.AIMG_BF16))
    monkeypatch.setattr(attention, "describe_pages", lambda k, v, table, lengths: _native.AimgPages(
        kv_heads=k.shape[1], page_size=k.shape[2], dim=k.shape[3], max_pages=table.shape[1]))
    return Recorder(monkeypatch, attention)


def test_the_workspaces_of_split_attention_live_until_their_launch(on_cpu):
    """A thread that allocates between the workspace and the launch must not be given the same memory."""
    q, k = (torch.zeros(n, 1, 64, dtype=torch.bfloat16) for n in (3, 4000))
    attention.prompt_attention(q, k, k, _ints(0, 3), _ints(0, 4000))
    work, nbytes = on_cpu.launches[-1][0][-2:]
    assert nbytes > 0 and on_cpu.living(work) is not None
    pages = torch.zeros(300, 1, 16, 64, dtype=torch.bfloat16)
    attention.tree_attention(q, pages, pages, _ints(*range(300)).view(1, 300), _ints(4000), _ints(0), _ints(0, 3), max_drafts=3)
    work, nbytes = on_cpu.launches[-1][0][-2:]
    assert nbytes > 0 and on_cpu.living(work) is not None
