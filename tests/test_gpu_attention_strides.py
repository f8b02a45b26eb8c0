"""Query rows far apart in memory, and one row of keys."""
import pytest
import torch

from afterimage_amd.runtime.attention import prompt_attention
from tests.test_gpu_prompt_attention import _case, _offsets
from tests.test_gpu_tree_attention import Case

pytestmark = pytest.mark.gpu

FAR = (1 << 24) + 8


def _apart(x):
    """x with its rows FAR elements apart."""
    wide = torch.empty(x.shape[0], FAR, dtype=x.dtype, device="cuda")
    y = wide.as_strided(x.shape, (FAR, x.shape[2], 1))
    y.copy_(x)
    return y


def test_prompt_rows():
    q, k, v = _case([5, 4], [5, 4], 4, 2, 64, torch.bfloat16)
    want = prompt_attention(q, k, v, _offsets([5, 4]))
    assert torch.equal(prompt_attention(_apart(q), k, v, _offsets([5, 4])), want)
    assert torch.equal(prompt_attention(q, k, v, _offsets([5, 4]), out=_apart(torch.zeros_like(q))), want)


def test_one_key():
    q, k, v = _case([1], [1], 4, 2, 64, torch.float16)
    assert torch.equal(prompt_attention(q, _apart(k), _apart(v), _offsets([1])), prompt_attention(q, k, v, _offsets([1])))


def test_drafted_rows():
    c = Case([45, 20], [3, 4], 8, 2, 128, 16, torch.bfloat16)
    assert torch.equal(c.run(q=_apart(c.q)), c.run())
