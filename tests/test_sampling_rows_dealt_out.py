"""Where a row's work is dealt out to several workgroups: by its length, its type and the number of rows."""
import ctypes

import pytest
import torch

from afterimage_amd import _native
from afterimage_amd.runtime.sampling import MAX_ROWS, MAX_VOCAB, sample


def _nbytes(rows, vocab):
    nbytes = ctypes.c_size_t(0)
    _native.check(_native.lib().aimg_sample_workspace_nbytes(rows, vocab, ctypes.byref(nbytes)))
    return nbytes.value


def test_longer_rows_are_dealt_out_where_there_are_more_of_them():
    """No number of rows at which all lengths end; none come back past it."""
    ends = []
    for vocab in (50001, 65536, 90001, 120000, 151936, 200000, MAX_VOCAB):
        dealt = [_nbytes(rows, vocab) > 0 for rows in range(1, 300)]
        end = sum(dealt)
        assert dealt == [i < end for i in range(299)]
        ends.append(end)
    assert ends[0] == 0 and ends[1] > 0 and sorted(set(ends)) == ends and ends[-1] > 64
    assert _nbytes(MAX_ROWS, MAX_VOCAB) == 0 and _nbytes(0, MAX_VOCAB) == 0


def test_too_little_workspace_is_refused_where_the_type_is_dealt_out():
    at, lib = 1 << 20, _native.lib()
    for rows, vocab, kind in ((1, MAX_VOCAB, _native.AIMG_BF16), (8, 65536, _native.AIMG_FP32), (90, MAX_VOCAB, _native.AIMG_FP32)):
        for work, nbytes in ((None, 1 << 30), (at, _nbytes(rows, vocab) - 1), (at + 4, 1 << 30)):
            assert lib.aimg_sample(at, rows, vocab, vocab, kind, at, _native.AimgSampling(), at, None, work, nbytes, None) == _native.AIMG_ERR_INVALID_ARGUMENT
            assert b"workspace" in lib.aimg_last_error()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,vocab,rows", [
    (torch.bfloat16, 72511, 1), (torch.bfloat16, 72512, 1), (torch.float32, 60426, 1), (torch.float32, 60427, 1),
    (torch.float16, 104767, 64), (torch.float16, 104768, 64), (torch.float16, 104768, 65), (torch.float32, 87306, 64), (torch.float32, 87307, 64),
    (torch.bfloat16, 140400, 65), (torch.bfloat16, 140399, 65), (torch.float32, 262144, 145), (torch.float32, 262144, 146)])
@pytest.mark.parametrize("own", [False, True])
def test_rows_on_both_sides(dtype, vocab, rows, own):
    """A row's token and its logarithm are the same bits as those of the row in a call of 256, which are not dealt out."""
    g = torch.Generator(device="cuda").manual_seed(vocab + rows)
    x = (torch.randn(rows, vocab, generator=g, device="cuda") * 2.5).to(dtype)
    u = torch.rand(rows, generator=g, device="cuda")
    settings = dict(temperature=0.8, top_k=300, top_p=0.95, min_p=0.001)
    if own:
        settings = {name: torch.full((rows,), value, dtype=torch.int32 if name == "top_k" else torch.float32, device="cuda") for name, value in settings.items()}
    got = sample(x, u, logprobs=True, **settings)
    assert _nbytes(256, vocab) == 0
    more = 256 - rows
    if own:
        settings = {name: torch.cat((value, value[:1].expand(more))) for name, value in settings.items()}
    want = sample(torch.cat((x, x[:1].expand(more, -1))), torch.cat((u, u[:1].expand(more))), logprobs=True, **settings)
    assert torch.equal(got[0], want[0][:rows]) and torch.equal(got[1], want[1][:rows])
