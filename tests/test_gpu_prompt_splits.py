"""Prompts split along their keys: where their parts lie, and many sequences a call."""
import ctypes
import random

import pytest
import torch

from afterimage_amd import _native
from afterimage_amd.runtime.attention import prompt_attention
from tests.attention_oracle import check
from tests.test_gpu_prompt_attention import _case, _expected, _offsets

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows,keys,heads,kv,dim", [
    # Sequences of one length, and some without keys to split between them.
    ([7] * 12, [2100] * 12, 8, 1, 128),
    ([7, 0, 7, 3] * 4, [2100, 900, 2100, 2] * 4, 8, 1, 64),
    # More than 64 sequences, the long ones at both ends and in the middle.
    ([40] + [1] * 70 + [9] + [2] * 70 + [130], [9000] + [1] * 70 + [30000] + [5] * 70 + [60000], 8, 1, 64),
    ([3] * 200, [700] * 199 + [9000], 1, 1, 64),
    # Long sequences whose rows in every part would pass the scratch planned: parts are made longer.
    ([1] * 10 + [600] + [1] * 10, [10] * 10 + [20000] + [10] * 10, 8, 1, 256),
    ([600, 600] + [1] * 20, [9000, 9000] + [10] * 20, 8, 1, 256),
    ([500, 300, 5, 400], [500, 6000, 9000, 700], 16, 2, 256),
])
def test_parts_of_several_sequences(rows, keys, heads, kv, dim):
    q, k, v = _case(rows, keys, heads, kv, dim, torch.bfloat16)
    lse = torch.empty(q.shape[:2], device="cuda")
    out = prompt_attention(q, k, v, _offsets(rows), _offsets(keys), lse=lse)
    o, bound, want = _expected(q, k, v, rows, keys, dim ** -0.5)
    check(out, o, bound)
    none = want == float("-inf")  # a row that sees no key
    assert torch.equal(lse == float("-inf"), none)
    assert (lse.double() - want)[~none].abs().max().item() <= 2.0 ** -24 * (3 * dim * 8 + 64)
    assert torch.equal(prompt_attention(q, k, v, _offsets(rows), _offsets(keys)), out)


@pytest.mark.parametrize("seed", range(3))
def test_many_short_sequences(seed):
    """Some 200 of them, empty ones among them: their place is searched for in more than one round."""
    rng = random.Random(seed)
    rows = [rng.choice((0, 1, rng.randint(1, 40), rng.randint(1, 150))) for _ in range(200 + seed)]
    keys = [n + rng.choice((0, 0, rng.randint(0, 90))) for n in rows]
    q, k, v = _case(rows, keys, 4, 2, 64, torch.float16, seed)
    out = prompt_attention(q, k, v, _offsets(rows), _offsets(keys))
    o, bound, _ = _expected(q, k, v, rows, keys, 64 ** -0.5)
    check(out, o, bound)


@pytest.mark.parametrize("q_offsets,k_offsets", [
    ([0, 20, 0, 20], [0, 6000, 0, 6000]),
    ([0, 20, 0, 20, -5, 999], [0, 6000, -9, 7000, 3, 6000]),
    ([20, 0, 20, 0, 20], [0, 6000, 6000, 0, 6000]),
])
def test_offsets_that_fall_stay_within_the_workspace(q_offsets, k_offsets):
    """Sequences over each other need more parts than were planned for: what lies past the workspace is not touched."""
    q, k, v = _case([20], [6000], 8, 1, 64, torch.bfloat16)
    out, n, seqs = torch.zeros_like(q), ctypes.c_size_t(), len(q_offsets) - 1
    lib = _native.lib()
    _native.check(lib.aimg_prompt_workspace_nbytes(20, 6000, 8, 1, 64, seqs, ctypes.byref(n)))
    assert n.value > 0
    guarded = torch.full((16 * n.value,), 77, dtype=torch.uint8, device="cuda")
    at = [torch.tensor(x, dtype=torch.int32, device="cuda") for x in (q_offsets, k_offsets)]
    heads = [_native.AimgHeads(x.data_ptr(), x.shape[0], *x.stride()[:2], *x.shape[1:]) for x in (q, k, v, out)]
    _native.check(lib.aimg_prompt_attention(*heads, at[0].data_ptr(), at[1].data_ptr(), seqs, _native.AIMG_BF16, 0.125, None,
                                            guarded.data_ptr(), n.value, torch.cuda.current_stream().cuda_stream))
    torch.cuda.synchronize()
    assert bool((guarded[n.value:] == 77).all())
