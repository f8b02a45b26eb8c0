"""Attention has no backward pass: what asks for a gradient is refused, not
answered without one. No GPU is used: launches are recorded, not made."""
import pytest
import torch

from afterimage_amd.runtime import attention, kv_cache
from tests.test_workspaces import _ints, on_cpu  # noqa: F401


def _prompt(**grad):
    q, k, v = (torch.zeros(3, 2, 64, dtype=torch.bfloat16, requires_grad=x in grad) for x in "qkv")
    return attention.prompt_attention(q, k, v, _ints(0, 3))


def _tree(**grad):
    q = torch.zeros(3, 2, 64, dtype=torch.bfloat16, requires_grad="q" in grad)
    k, v = (torch.zeros(4, 2, 16, 64, dtype=torch.bfloat16, requires_grad=x in grad) for x in "kv")
    return attention.tree_attention(q, k, v, _ints(0, 1, 2, 3).view(1, 4), _ints(20), _ints(0), _ints(0, 3), max_drafts=3)


@pytest.mark.parametrize("call", [_prompt, _tree])
@pytest.mark.parametrize("which", ["q", "k", "v"])
def test_inputs_that_require_a_gradient_are_refused(on_cpu, call, which):  # noqa: F811
    with pytest.raises(RuntimeError, match="no backward"):
        call(**{which: True})
    assert not on_cpu.launches
    with torch.no_grad():
        assert not call(**{which: True}).requires_grad
    with torch.inference_mode():
        call(**{which: True})
    assert len(on_cpu.launches) == 2


def test_rows_that_require_a_gradient_are_not_appended():
    c = object.__new__(kv_cache.PagedKVCache)
    c._index, c.kv_heads, c.dim, c.pool = -1, 2, 64, torch.zeros(0, dtype=torch.bfloat16)
    rows = torch.zeros(3, 2, 64, dtype=torch.bfloat16, requires_grad=True)
    with pytest.raises(RuntimeError, match="no backward"):
        c._rows(rows, "k")
    with torch.no_grad():
        assert c._rows(rows, "k").n_rows == 3
