"""What turns, stores, reads, attends over and samples refuses bad calls before
anything is launched (no GPU is used: nothing here gets as far as a launch)."""
import ctypes

import pytest
import torch

from afterimage_amd import _native
from afterimage_amd.runtime import attention, kv_cache, sampling

BAD, UNSUPPORTED, OK = _native.AIMG_ERR_INVALID_ARGUMENT, _native.AIMG_ERR_UNSUPPORTED, _native.AIMG_OK
AT = 1 << 20


def _heads(n=4, heads=2, dim=64, data=AT, row=None, head=None):
    return _native.AimgHeads(data, n, heads * dim if row is None else row, dim if head is None else head, heads, dim)


def _cache(**more):
    c = _native.AimgCache(AT, AT, AT, AT, AT, AT, 2, 10, 2, 16, 64, 3, 8)
    for name, value in more.items():
        setattr(c, name, value)
    return c


def _rotary(cos=AT, sin=AT, n=100, half=32, interleaved=0):
    return _native.AimgRotary(cos, sin, n, half, interleaved)


def _append(cache=None, scales=None, layer=0, q="", k=None, v=None, out=None, seqs=AT, offsets=AT, n=1, rotary="", kind=0):
    q = _heads(heads=4) if q == "" else q
    return _native.lib().aimg_cache_append_rotated(cache or _cache(), scales, layer, q, k or _heads(), v or k or _heads(), out or q, seqs, offsets, n,
                                                   _rotary() if rotary == "" else rotary, None, kind, None)


@pytest.mark.parametrize("args,code,message", [
    (dict(cache=_cache(n_layers=0)), BAD, b"every size"), (dict(cache=_cache(pool=None)), BAD, b"null"), (dict(layer=2), BAD, b"layer"),
    (dict(layer=-1), BAD, b"layer"), (dict(k=_heads(heads=3)), BAD, b"k must have 2 heads"), (dict(v=_heads(dim=32)), BAD, b"v must have"),
    (dict(v=_heads(n=5)), BAD, b"same rows"), (dict(q=_heads(n=5, heads=4)), BAD, b"same rows"), (dict(q=_heads(heads=4, dim=32)), BAD, b"q must have"),
    (dict(out=_heads(heads=3)), BAD, b"q_out must have"), (dict(k=_heads(data=None)), BAD, b"null data"), (dict(k=_heads(data=AT + 8)), UNSUPPORTED, b"aligned"),
    (dict(k=_heads(row=132)), UNSUPPORTED, b"16 bytes"), (dict(q=_heads(heads=4, head=-64)), UNSUPPORTED, b"negative"), (dict(k=_heads(n=-1)), BAD, b"n_rows"),
    (dict(n=-1), BAD, b"n_seqs"), (dict(n=9000), UNSUPPORTED, b"8192"), (dict(seqs=None), BAD, b"null"), (dict(kind=2), UNSUPPORTED, b"type"),
    (dict(rotary=_rotary(cos=None)), BAD, b"rotary"), (dict(rotary=_rotary(n=0)), BAD, b"positions"), (dict(rotary=_rotary(half=0)), BAD, b"half"),
    (dict(rotary=_rotary(half=33)), BAD, b"half"), (dict(rotary=_rotary(sin=AT + 2)), UNSUPPORTED, b"4-byte"),
    (dict(cache=_cache(dim=264), k=_heads(dim=264), q=_heads(heads=4, dim=264)), UNSUPPORTED, b"at most 256"),
    (dict(cache=_cache(dim=72), scales=AT), UNSUPPORTED, b"multiple of 16"), (dict(cache=_cache(page_size=24), scales=AT), UNSUPPORTED, b"page_size"),
    (dict(scales=AT + 2), UNSUPPORTED, b"4-byte"), (dict(cache=_cache(dim=272), scales=AT), UNSUPPORTED, b"up to 256"),
    (dict(q=None, k=_heads(n=(1 << 31) - 9), n=1, scales=AT), UNSUPPORTED, b"too many rows"),
    (dict(q=_heads(n=1 << 24, heads=4), k=_heads(n=1 << 24)), UNSUPPORTED, b"too many rows"),
])
def test_append_rotated_refuses(args, code, message):
    assert _append(**args) == code
    assert message in _native.lib().aimg_last_error()


def test_nothing_to_do_is_no_error():
    lib = _native.lib()
    assert _append(n=0) == OK and _append(q=_heads(n=0, heads=4), k=_heads(n=0)) == OK and _append(q=None, n=0, scales=AT, rotary=None) == OK
    assert lib.aimg_cache_read(_cache(), None, 0, AT, AT, None, 0, _heads(), _heads(), 0, None) == OK
    assert lib.aimg_cache_read(_cache(), AT, 0, AT, AT, None, 1, _heads(n=0), _heads(n=0), 0, None) == OK
    for entry in (lib.aimg_cache8_fork, ):
        assert entry(_cache(), AT, AT, AT, 0, None, 0, None) == OK
    assert lib.aimg_cache8_commit(_cache(), AT, AT, AT, 4, AT, 0, AT, None) == OK
    assert lib.aimg_sample(None, 0, 10, 10, 0, None, _native.AimgSampling(), None, None, None, 0, None) == OK
    assert _tree8(n=0) == OK


@pytest.mark.parametrize("args,code,message", [
    (dict(layer=5), BAD, b"layer"), (dict(k=_heads(heads=1)), BAD, b"k must have"), (dict(v=_heads(n=3)), BAD, b"same rows"), (dict(kind=7), UNSUPPORTED, b"type"),
    (dict(k=_heads(row=4)), UNSUPPORTED, b"16 bytes"), (dict(scales=AT, cache=_cache(page_size=8)), UNSUPPORTED, b"page_size"), (dict(n=-2), BAD, b"n_seqs"),
    (dict(k=_heads(n=(1 << 27) + 1), v=_heads(n=(1 << 27) + 1)), UNSUPPORTED, b"too many rows"),
])
def test_read_refuses(args, code, message):
    a = dict(cache=_cache(), scales=None, layer=0, k=_heads(), v=_heads(), n=1, kind=0) | args
    assert _native.lib().aimg_cache_read(a["cache"], a["scales"], a["layer"], AT, AT, None, a["n"], a["k"], a["v"], a["kind"], None) == code
    assert message in _native.lib().aimg_last_error()


def test_steps_of_eight_bits_refuse():
    lib = _native.lib()
    for call in (lambda s, c: lib.aimg_cache8_fork(c, s, AT, AT, 1, AT, 1 << 20, None),
                 lambda s, c: lib.aimg_cache8_commit(c, s, AT, AT, 4, AT, 1, AT, None),
                 lambda s, c: lib.aimg_cache8_compact(c, s, AT, AT, AT, AT, 1 << 20, None)):
        assert call(None, _cache()) == BAD and b"scales" in lib.aimg_last_error()
        assert call(AT, _cache(dim=24)) == UNSUPPORTED and b"multiple of 16" in lib.aimg_last_error()
        assert call(AT, _cache(page_size=20)) == UNSUPPORTED
    assert lib.aimg_cache8_fork(_cache(), AT, AT, AT, 3, AT, 4, None) == BAD and b"workspace" in lib.aimg_last_error()
    assert lib.aimg_cache8_commit(_cache(), AT, AT, AT, -1, AT, 1, AT, None) == BAD
    assert lib.aimg_cache8_compact(_cache(), AT, AT, AT, None, AT, 1 << 20, None) == BAD


def _pages(**more):
    p = _native.AimgPages(AT, AT, AT, AT, 2 * 16 * 64, 64, 16 * 64, 8, 10, 16, 2, 64, 3, 8)
    for name, value in more.items():
        setattr(p, name, value)
    return p


def _tree8(q=None, pages=None, scales="", n=1, kind=0):
    q = q or _heads()
    scales = _native.AimgPageScales(AT, AT, 2, 1) if scales == "" else scales
    return _native.lib().aimg_tree8_attention(q, pages or _pages(), scales, q, AT, AT, n, None, 0, 1, 10, kind, 1.0, None, None, 0, None)


@pytest.mark.parametrize("args,code,message", [
    (dict(scales=None), BAD, b"scales"), (dict(scales=_native.AimgPageScales(None, AT, 2, 1)), BAD, b"null"),
    (dict(scales=_native.AimgPageScales(AT, AT + 1, 2, 1)), UNSUPPORTED, b"4-byte"), (dict(scales=_native.AimgPageScales(AT, AT, -2, 1)), UNSUPPORTED, b"negative"),
    (dict(pages=_pages(dim=72), q=_heads(dim=72)), UNSUPPORTED, b"multiple of 16"), (dict(pages=_pages(page_size=8)), UNSUPPORTED, b"page_size"),
    (dict(pages=_pages(slot_stride=72)), UNSUPPORTED, b"16 bytes"), (dict(kind=2), UNSUPPORTED, b"type"), (dict(q=_heads(dim=32)), BAD, b"dim"),
])
def test_attention_over_eight_bits_refuses(args, code, message):
    assert _tree8(**args) == code
    assert message in _native.lib().aimg_last_error()


@pytest.mark.parametrize("args,code,message", [
    (dict(rows=-1), BAD, b"n_rows"), (dict(vocab=0), BAD, b"vocab"), (dict(vocab=(1 << 18) + 1), UNSUPPORTED, b"2^18"), (dict(rows=(1 << 21) + 1), UNSUPPORTED, b"2^21"), (dict(stride=-1), BAD, b"row_stride"),
    (dict(kind=3), UNSUPPORTED, b"type"), (dict(logits=None), BAD, b"null"), (dict(uniforms=None), BAD, b"null"), (dict(tokens=None), BAD, b"null"),
    (dict(settings=None), BAD, b"settings"), (dict(logits=AT + 1), UNSUPPORTED, b"aligned"), (dict(tokens=AT + 4), UNSUPPORTED, b"aligned"),
    (dict(logits=AT + 2, kind=2), UNSUPPORTED, b"aligned"), (dict(vocab=100000), BAD, b"workspace"), (dict(vocab=100000, work=AT, nbytes=100), BAD, b"workspace"),
    (dict(vocab=100000, work=AT + 4, nbytes=1 << 20), BAD, b"workspace"),
])
def test_sample_refuses(args, code, message):
    a = dict(logits=AT, rows=2, stride=10, vocab=10, kind=0, uniforms=AT, settings=_native.AimgSampling(), tokens=AT, work=None, nbytes=0) | args
    assert _native.lib().aimg_sample(a["logits"], a["rows"], a["stride"], a["vocab"], a["kind"], a["uniforms"], a["settings"], a["tokens"], None, a["work"], a["nbytes"],
                                     None) == code
    assert message in _native.lib().aimg_last_error()


def test_calls_from_python_run_on_the_gpu_only():
    x = torch.zeros(2, 10)
    with pytest.raises(RuntimeError, match="GPU only"):
        sampling.sample(x, torch.zeros(2))
    with pytest.raises(RuntimeError, match="GPU only"):
        kv_cache.PagedKVCache.allocate(1, 2, 16, 1, 16, 1, 1, torch.float8_e4m3fn, "cpu")
    for args in ((0, 16), (4, 0), (4, 3), (4, 16, 0.0)):
        with pytest.raises(ValueError, match="rotary_tables"):
            attention.rotary_tables(*args, device="cpu")


def test_rotary_tables():
    cos, sin = attention.rotary_tables(5, 4, 100.0, "cpu")
    assert cos.shape == sin.shape == (5, 2) and cos.dtype is torch.float32
    angle = torch.arange(5, dtype=torch.float64)[:, None] * torch.tensor([1.0, 0.1], dtype=torch.float64)
    assert torch.equal(cos, angle.cos().float()) and torch.equal(sin, angle.sin().float())
