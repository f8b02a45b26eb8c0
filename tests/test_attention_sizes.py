"""What the attention calls ask of a caller's memory, and the sizes they take (no GPU is used)."""
import ctypes

import pytest

from afterimage_amd import _native


def _prompt_nbytes(*sizes):
    n = ctypes.c_size_t()
    assert _native.lib().aimg_prompt_workspace_nbytes(*sizes, ctypes.byref(n)) == _native.AIMG_OK
    return n.value


@pytest.mark.parametrize("seqs", [1, 2, 3, 8, 16, 24, 32, 64, 200, 256])
@pytest.mark.parametrize("heads,kv,dim", [(8, 1, 128), (40, 8, 128), (8, 1, 256), (4, 4, 64), (64, 1, 128)])
def test_split_prompts_need_little_scratch_however_many_they_are(seqs, heads, kv, dim):
    """512 workgroups of 128 rows run at a time: parts of twice as many, or 64 MiB, are the most."""
    row = 4 * (64 if dim <= 64 else 128 if dim <= 128 else 256) + 8
    most = max(64 << 20, 2 * 2 * 512 * 128 * row)
    sizes = [(seqs * n, seqs * m, heads, kv, dim, seqs) for n in (1, 7, 40, 112, 600) for m in (600, 2112, 9000, 64000, 1 << 20)
             if seqs * m < 1 << 31]
    for size in sizes:
        assert _prompt_nbytes(*size) <= most, size
    # A single sequence's parts are known exactly: a row of sums and two numbers for each row, head and part.
    if seqs == 1:
        assert all(_prompt_nbytes(*size) % (size[0] * heads * row) == 0 for size in sizes)
