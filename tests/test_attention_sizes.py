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


def _heads(n=4, heads=2, dim=64, data=1 << 20, row=None, head=None):
    return _native.AimgHeads(data, n, heads * dim if row is None else row, dim if head is None else head, heads, dim)


def test_keys_whose_tiles_would_pass_32_bits_are_refused():
    """The first key of a tile and the tile's 64 stay below 2^31."""
    lib, n = _native.lib(), ctypes.c_size_t()
    for rows, prompt, nbytes in [((1 << 31) - 65, b"null offsets", _native.AIMG_OK), ((1 << 31) - 64, b"2^31 - 64", _native.AIMG_ERR_UNSUPPORTED),
                                 ((1 << 31) - 1, b"2^31 - 64", _native.AIMG_ERR_UNSUPPORTED)]:
        q, k = _heads(), _heads(n=rows, row=0)
        assert lib.aimg_prompt_attention(q, k, k, q, None, None, 1, 0, 1.0, None, None, 0, None) != _native.AIMG_OK
        assert prompt in lib.aimg_last_error(), rows
        assert lib.aimg_prompt_workspace_nbytes(4, rows, 2, 2, 64, 1, ctypes.byref(n)) == nbytes, rows


@pytest.mark.parametrize("page_size", [1 << 28, (1 << 29) + (1 << 28), (1 << 30) - 1])
def test_pages_whose_bytes_pass_64_bits_are_refused(page_size):
    lib = _native.lib()
    c = _native.AimgCache(1 << 20, 1 << 20, 1 << 20, 1 << 20, 1 << 20, 1 << 20, 1, 1, 1 << 20, page_size, 8 * 1023, 1, 1)
    assert lib.aimg_cache_reserve(c, None, None, 0, None) == _native.AIMG_ERR_UNSUPPORTED
    assert b"2^31 bytes" in lib.aimg_last_error()


def test_query_rows_may_be_any_distance_apart():
    """Only rows of keys and values are read many at a time, by 32-bit offsets; a single row has no distance."""
    lib = _native.lib()
    far = (1 << 24) + 8
    for q, k, message in [(_heads(row=1 << 40), _heads(), b"null offsets"), (_heads(), _heads(n=1, row=far), b"null offsets"),
                          (_heads(), _heads(row=1 << 24), b"null offsets"), (_heads(), _heads(row=far), b"2^24")]:
        assert lib.aimg_prompt_attention(q, k, k, q, None, None, 1, 0, 1.0, None, None, 0, None) != _native.AIMG_OK
        assert message in lib.aimg_last_error()
