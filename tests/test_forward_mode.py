"""No call has a derivative in forward mode: an input with a tangent is refused, not answered without one. No GPU is used:
launches are recorded, not made."""
import pytest
import torch
from torch.autograd import forward_ad

from afterimage_amd.runtime import attention, kv_cache, sampling
from tests.test_attention_gradients import _ints
from tests.test_workspaces import on_cpu  # noqa: F401


def _dual(x):
    return forward_ad.make_dual(x, torch.ones_like(x))


def _prompt(which):
    inputs = [torch.zeros(3, 2, 64, dtype=torch.bfloat16) for _ in range(3)]
    if which:
        inputs["qkv".index(which)] = _dual(inputs["qkv".index(which)])
    return attention.prompt_attention(*inputs, _ints(0, 3))


def _tree(which):
    inputs = [torch.zeros(3, 2, 64, dtype=torch.bfloat16)] + [torch.zeros(4, 2, 16, 64, dtype=torch.bfloat16) for _ in range(2)]
    if which:
        inputs["qkv".index(which)] = _dual(inputs["qkv".index(which)])
    return attention.tree_attention(*inputs, _ints(0, 1, 2, 3).view(1, 4), _ints(20), _ints(0), _ints(0, 3), max_drafts=3)


@pytest.mark.parametrize("call", [_prompt, _tree])
@pytest.mark.parametrize("which", ["q", "k", "v"])
def test_inputs_with_a_tangent_are_refused(on_cpu, call, which):  # noqa: F811
    with forward_ad.dual_level():
        with pytest.raises(RuntimeError, match="%s(_pages)? has a tangent" % which):
            call(which)
        with torch.no_grad(), pytest.raises(RuntimeError, match="tangent"):  # which records no gradients, and tangents all the same
            call(which)
        assert not on_cpu.launches
        call(None)
        with torch.inference_mode():
            call(which)
    assert len(on_cpu.launches) == 2


def test_rows_with_a_tangent_are_not_appended():
    c = object.__new__(kv_cache.PagedKVCache)
    c._index, c.kv_heads, c.dim, c.pool = -1, 2, 64, torch.zeros(0, dtype=torch.bfloat16)
    rows = torch.zeros(3, 2, 64, dtype=torch.bfloat16)
    with forward_ad.dual_level():
        with pytest.raises(RuntimeError, match="k has a tangent"):
            c._rows(_dual(rows), "k")
        assert c._rows(rows, "k").n_rows == 3


@pytest.mark.parametrize("which", ["cos", "sin"])
def test_tables_with_a_tangent_are_refused(which, monkeypatch):
    made = []
    monkeypatch.setattr(kv_cache, "launch", lambda *args: made.append(args))
    c = object.__new__(kv_cache.PagedKVCache)
    c._index, c.kv_heads, c.dim, c.n_layers, c._cache, c._scales_at = -1, 2, 64, 1, None, None
    c.pool, c._lib = torch.zeros(0, dtype=torch.bfloat16), type("Lib", (), {"aimg_cache_append_rotated": None})
    x, tables = torch.zeros(3, 2, 64, dtype=torch.bfloat16), {"cos": torch.zeros(8, 32), "sin": torch.zeros(8, 32)}
    with forward_ad.dual_level():
        c.append_rotated(0, x, x, x, _ints(0), _ints(0, 3), **tables)
        assert len(made) == 1
        tables[which] = _dual(tables[which])
        with pytest.raises(RuntimeError, match="%s has a tangent" % which):
            c.append_rotated(0, x, x, x, _ints(0), _ints(0, 3), **tables)
    assert len(made) == 1


@pytest.mark.gpu
def test_logits_and_settings_with_a_tangent_are_refused():
    x, u, t = torch.zeros(2, 10, device="cuda"), torch.zeros(2, device="cuda"), torch.ones(2, device="cuda")
    with forward_ad.dual_level():
        with pytest.raises(RuntimeError, match="logits has a tangent"):
            sampling.sample(_dual(x), u, logprobs=True)
        with pytest.raises(RuntimeError, match="temperature has a tangent"):
            sampling.sample(x, u, temperature=_dual(t), logprobs=True)
        assert sampling.sample(x, u, temperature=t).tolist() == [0, 0]
