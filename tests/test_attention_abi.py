"""The attention and cache entry points refuse what they cannot serve before
anything is launched (no GPU is used: nothing here gets as far as a launch)."""
import ctypes

import pytest
import torch

from afterimage_amd import _native
from afterimage_amd.runtime import attention, kv_cache

BAD, UNSUPPORTED, OK = _native.AIMG_ERR_INVALID_ARGUMENT, _native.AIMG_ERR_UNSUPPORTED, _native.AIMG_OK


def _heads(n=4, heads=2, dim=64, data=1 << 20, row=None, head=None):
    return _native.AimgHeads(data, n, heads * dim if row is None else row, dim if head is None else head, heads, dim)


def _pages(**more):
    p = _native.AimgPages(1 << 20, 1 << 20, 1 << 20, 1 << 20, 2 * 16 * 64, 64, 16 * 64, 8, 10, 16, 2, 64, 3, 8)
    for name, value in more.items():
        setattr(p, name, value)
    return p


def _cache(**more):
    c = _native.AimgCache(1 << 20, 1 << 20, 1 << 20, 1 << 20, 1 << 20, 1 << 20, 2, 10, 2, 16, 64, 3, 8)
    for name, value in more.items():
        setattr(c, name, value)
    return c


def _prompt(q=None, k=None, v=None, out=None, at=64, n=1, kind=0, scale=1.0):
    q, k = q or _heads(), k or _heads()
    v, out = v or k, out or q
    return _native.lib().aimg_prompt_attention(q, k, v, out, at, at, n, kind, scale, None, None, 0, None)


def _tree(q=None, pages=None, n=1, most=1, context=10, words=1, scale=1.0, at=64, kind=0, work=None, nbytes=0):
    q = q or _heads()
    return _native.lib().aimg_tree_attention(q, pages or _pages(), q, at, at, n, 64, words, most, context, kind, scale, None, work,
                                             nbytes, None)


@pytest.mark.parametrize("args,code,message", [
    (dict(q=_heads(dim=60)), UNSUPPORTED, b"multiple of 8"), (dict(q=_heads(dim=264)), UNSUPPORTED, b"256"),
    (dict(q=_heads(data=None)), BAD, b"null"), (dict(q=_heads(data=(1 << 20) + 2)), UNSUPPORTED, b"aligned"),
    (dict(k=_heads(row=129)), UNSUPPORTED, b"aligned"), (dict(k=_heads(row=-128)), UNSUPPORTED, b"negative"),
    (dict(k=_heads(row=1 << 25)), UNSUPPORTED, b"2^24"), (dict(k=_heads(heads=3)), BAD, b"multiple of k"),
    (dict(k=_heads(dim=128)), BAD, b"dim"), (dict(v=_heads(n=5)), BAD, b"same rows"), (dict(out=_heads(n=5)), BAD, b"q's shape"),
    (dict(scale=0.0), BAD, b"scale"), (dict(scale=float("inf")), BAD, b"scale"), (dict(n=-1), BAD, b"n_seqs"),
    (dict(at=None), BAD, b"offsets"), (dict(kind=2), UNSUPPORTED, b"type"), (dict(q=_heads(n=-1)), BAD, b"n_rows"),
])
def test_prompt_attention_refuses(args, code, message):
    assert _prompt(**args) == code
    assert message in _native.lib().aimg_last_error()


def test_nothing_to_do_is_no_error():
    lib = _native.lib()
    assert _prompt(n=0, at=None) == OK
    assert _prompt(q=_heads(n=0, data=None)) == OK
    assert _tree(n=0, at=None) == OK
    assert lib.aimg_tree_masks(None, None, 0, 0, 1, None, None) == OK
    c = _cache()
    assert lib.aimg_cache_reserve(c, None, None, 0, None) == OK
    assert lib.aimg_cache_release(c, None, 0, None) == OK
    assert lib.aimg_cache_fork(c, None, None, 0, None, 0, None) == OK
    assert lib.aimg_cache_append(c, 0, _heads(n=0, data=None), _heads(n=0, data=None), 64, 64, 1, None) == OK


@pytest.mark.parametrize("args,code,message", [
    (dict(pages=_pages(n_pages=0)), BAD, b"at least 1"), (dict(pages=_pages(page_size=1 << 28)), UNSUPPORTED, b"2^30"),
    (dict(pages=_pages(k=None)), BAD, b"null"), (dict(pages=_pages(slot_stride=60)), UNSUPPORTED, b"aligned"),
    (dict(pages=_pages(k=(1 << 20) + 8)), UNSUPPORTED, b"aligned"), (dict(pages=_pages(dim=128)), BAD, b"dim"),
    (dict(pages=_pages(kv_heads=3)), BAD, b"multiple of their heads"), (dict(most=0), BAD, b"max_drafts"),
    (dict(context=-1), BAD, b"max_context"), (dict(context=1 << 31), BAD, b"max_context"), (dict(words=0), BAD, b"mask_words"),
    (dict(at=None), BAD, b"null seqs"), (dict(context=1 << 20), BAD, b"workspace"), (dict(kind=-1, context=0), UNSUPPORTED, b"type"),
])
def test_tree_attention_refuses(args, code, message):
    assert _tree(**args) == code
    assert message in _native.lib().aimg_last_error()


def test_tree_workspace_follows_the_sizes():
    lib, n = _native.lib(), ctypes.c_size_t()

    def nbytes(*sizes):
        assert lib.aimg_tree_workspace_nbytes(*sizes, ctypes.byref(n)) == OK
        return n.value
    assert nbytes(1, 40, 8, 128, 1, 1, 0) == 0
    # A row of padded sums and two numbers for each part of a row and head.
    parts, rest = divmod(nbytes(1, 40, 8, 128, 1, 1, 8000), 40 * (4 * 128 + 8))
    assert parts > 1 and rest == 0
    assert nbytes(3, 40, 8, 96, 1, 3, 8000) % (3 * 40 * (4 * 128 + 8)) == 0
    assert nbytes(0, 40, 8, 128, 0, 1, 8000) == 0
    assert lib.aimg_tree_workspace_nbytes(1, 40, 7, 128, 1, 1, 0, ctypes.byref(n)) == BAD
    assert lib.aimg_tree_workspace_nbytes(1, 40, 8, 128, 1, 1, 0, None) == BAD


def test_tree_sizes_at_their_limits():
    """Contexts past what a sequence can hold plan no part past it, drafts past the rows no rows; sizes whose product is too large are refused."""
    lib, n = _native.lib(), ctypes.c_size_t()

    def nbytes(*sizes):
        rc = lib.aimg_tree_workspace_nbytes(*sizes, ctypes.byref(n))
        return n.value if rc == OK else rc

    most = nbytes(1, 8, 8, 64, 1, 1, (1 << 30) - 1)
    assert most > 0 and most == nbytes(1, 8, 8, 64, 1, 1, (1 << 31) - 1) == nbytes(1, 8, 8, 64, 1, (1 << 31) - 1, (1 << 31) - 1)
    parts = most // (8 * (4 * 64 + 8))
    assert (parts - 1) * 8192 < 1 << 30
    assert nbytes(7, 40, 8, 64, 2, (1 << 31) - 1, 0) == nbytes(7, 40, 8, 64, 2, 7, 0)
    for sizes in [(1 << 30, 8, 8, 64, 1, 1, 0), (1, 1 << 20, 1 << 20, 64, 1 << 20, 1, 0), (64, 1 << 20, 1, 64, 1 << 18, 64, 0),
                  (1, 8, 8, 64, 1 << 20, 1, (1 << 30) - 1)]:
        assert nbytes(*sizes) == UNSUPPORTED, sizes


def test_prompt_workspace_follows_the_sizes():
    lib, n = _native.lib(), ctypes.c_size_t()

    def nbytes(*sizes):
        assert lib.aimg_prompt_workspace_nbytes(*sizes, ctypes.byref(n)) == OK
        return n.value
    # Rows that fill the GPU, or few keys: none. Few rows over many keys: a row of sums and two numbers a part.
    assert nbytes(16384, 16384, 40, 8, 128, 1) == 0 and nbytes(77, 77, 16, 16, 64, 1) == 0 and nbytes(0, 0, 4, 2, 64, 0) == 0
    parts, rest = divmod(nbytes(13, 8000, 8, 1, 96, 1), 13 * 8 * (4 * 128 + 8))
    assert parts > 1 and rest == 0
    assert lib.aimg_prompt_workspace_nbytes(13, 8000, 8, 3, 96, 1, ctypes.byref(n)) == BAD
    q, k = _heads(n=13, heads=8), _heads(n=8000, heads=1)
    assert lib.aimg_prompt_attention(q, k, k, q, 64, 64, 1, 0, 1.0, None, None, 0, None) == BAD
    assert b"workspace" in lib.aimg_last_error()


@pytest.mark.parametrize("more,code,message", [
    (dict(n_layers=0), BAD, b"at least 1"), (dict(n_pages=1 << 20), UNSUPPORTED, b"2^20"), (dict(dim=20), UNSUPPORTED, b"multiple of 8"),
    (dict(max_pages=1 << 28), UNSUPPORTED, b"2^30"), (dict(lengths=None), BAD, b"null"), (dict(pool=(1 << 20) + 8), UNSUPPORTED, b"aligned"),
    (dict(pool=None), BAD, b"null"), (dict(kv_heads=1 << 20, page_size=1 << 10), UNSUPPORTED, b"2^31"),
])
def test_cache_calls_refuse_a_bad_cache(more, code, message):
    lib, c = _native.lib(), _cache(**more)
    assert lib.aimg_cache_fork(c, 64, 64, 1, 64, 1 << 20, None) == code
    assert message in lib.aimg_last_error()
    assert lib.aimg_cache_commit(c, 64, 64, 1, 64, 1, 64, None) == code
    assert lib.aimg_cache_compact(c, 64, 64, 64, 64, 1 << 20, None) == code
    assert lib.aimg_cache_append(c, 0, _heads(dim=c.dim), _heads(dim=c.dim), 64, 64, 1, None) == code


def test_cache_calls_refuse_their_arguments():
    lib, c = _native.lib(), _cache()
    for rc, code, message in [
        (lambda: lib.aimg_cache_reserve(c, None, 64, 1, None), BAD, b"null"),
        (lambda: lib.aimg_cache_reserve(c, 64, 64, 8193, None), UNSUPPORTED, b"8192"),
        (lambda: lib.aimg_cache_release(c, 64, -1, None), BAD, b"n_seqs"),
        (lambda: lib.aimg_cache_append(c, 2, _heads(), _heads(), 64, 64, 1, None), BAD, b"layer"),
        (lambda: lib.aimg_cache_append(c, 0, _heads(heads=3), _heads(), 64, 64, 1, None), BAD, b"heads"),
        (lambda: lib.aimg_cache_append(c, 0, _heads(row=130), _heads(), 64, 64, 1, None), UNSUPPORTED, b"aligned"),
        (lambda: lib.aimg_cache_fork(c, 64, 64, 2, 64, 4 * 2 * 10 - 1, None), BAD, b"workspace"),
        (lambda: lib.aimg_cache_fork(c, 64, 64, 2, None, 1 << 20, None), BAD, b"workspace"),
        (lambda: lib.aimg_cache_commit(c, 64, 64, -1, 64, 1, 64, None), BAD, b"max_accepted"),
        (lambda: lib.aimg_cache_commit(c, 64, None, 1, 64, 1, 64, None), BAD, b"accepted"),
        (lambda: lib.aimg_cache_compact(c, 64, 64, 64, 64, 4 * 31 - 1, None), BAD, b"workspace"),
        (lambda: lib.aimg_cache_compact(c, None, 64, 64, 64, 1 << 20, None), BAD, b"new_table"),
        (lambda: lib.aimg_tree_masks(None, 64, 1, 4, 1, 64, None), BAD, b"null"),
        (lambda: lib.aimg_tree_masks(64, 64, 1, 4, 0, 64, None), BAD, b"mask_words"),
    ]:
        assert rc() == code, message
        assert message in lib.aimg_last_error()


def test_cpu_tensors_are_refused():
    x = torch.zeros(2, 2, 64, dtype=torch.bfloat16)
    at = torch.tensor([0, 2], dtype=torch.int32)
    with pytest.raises(RuntimeError, match="GPU only"):
        attention.prompt_attention(x, x, x, at)
    with pytest.raises(RuntimeError, match="GPU only"):
        attention.tree_masks(at, at, 2)
    with pytest.raises(RuntimeError, match="GPU only"):
        kv_cache.PagedKVCache.allocate(1, 4, 4, 2, 64, 2, 2, device="cpu")
