"""What attention over a cache asks for, found before anything is launched (no GPU is used)."""
import pytest
import torch

from afterimage_amd import _native
from afterimage_amd.runtime import kv_cache
from tests.test_workspaces import _ints, on_cpu  # noqa: F401


@pytest.fixture
def cache():
    c = object.__new__(kv_cache.PagedKVCache)
    c.n_layers, c._index, c.pool = 1, -1, torch.zeros(1, 2, 2, 2, 16, 64, dtype=torch.bfloat16)
    pages = _native.AimgPages(kv_heads=2, page_size=16, dim=64, max_pages=2)
    c._described = [(pages, None)]
    return c


def test_a_missing_max_drafts_is_named(cache, on_cpu, monkeypatch):  # noqa: F811
    monkeypatch.setattr(kv_cache, "_query", lambda q: (_native.AimgHeads(0, 1, 128, 64, 2, 64), -1, _native.AIMG_BF16))
    q = torch.zeros(1, 2, 64, dtype=torch.bfloat16)
    for options in ({}, {"max_context": 30}):
        with pytest.raises(TypeError, match="max_drafts"):
            cache.attend(0, q, _ints(0), _ints(0, 1), **options)
    with pytest.raises(TypeError):  # by name alone
        cache.attend(0, q, _ints(0), _ints(0, 1), None, 1)
    with pytest.raises(ValueError, match="max_drafts"):
        cache.attend(0, q, _ints(0), _ints(0, 1), max_drafts=0)
    assert not on_cpu.launches
    cache.attend(0, q, _ints(0), _ints(0, 1), max_drafts=1, max_context=30)
    assert len(on_cpu.launches) == 1
