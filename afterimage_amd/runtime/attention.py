"""Attention between a decoder layer's projections: whole prompts, and drafted
tokens over a paged cache.

The reference leaves attention to the model's own forward pass
(afterimage/runtime/streaming_engine.py:2154-2213 drives it); these are the
products a program runs between the q/k/v projections whose weights it decodes
and the output projection. Elements are bf16 or fp16; scores, softmax
statistics and sums are fp32. Work is ordered on the current stream and nothing
here synchronises. There is no backward pass: inputs that require a gradient are
refused while gradients are recorded.
"""
from __future__ import annotations

import ctypes
import functools
import math

import torch

from .. import _native

MAX_DIM = 256

_current_device = torch._C._cuda_getDevice
_stream_handle = torch._C._cuda_getCurrentRawStream

_TYPES = {torch.bfloat16: _native.AIMG_BF16, torch.float16: _native.AIMG_FP16}


# The calls are short (a few microseconds of GPU time for one token), so the
# checks go by the cheapest question first: a device's index rather than the
# device, shapes and strides taken apart once, descriptors built once a call.

def forward_only(x: torch.Tensor, name: str) -> None:
    """Refuses a tensor whose gradient autograd would expect."""
    if x.requires_grad and torch.is_grad_enabled():
        raise RuntimeError("%s requires a gradient, and attention has no backward pass: detach it, or call under torch.no_grad()" % name)


def _heads(x: torch.Tensor, name: str, dtype: torch.dtype, index: int, unit: int = 8) -> _native.AimgHeads:
    """The descriptor of rows of heads [n, heads, dim] of this type on GPU
    ``index``, any row and head strides that keep whole pieces of ``unit``
    elements aligned."""
    if x.get_device() != index or x.dtype is not dtype or x.dim() != 3:
        _refuse(x, name, dtype, index)
    n, heads, dim = x.shape
    row, head, one = x.stride()
    at = x.data_ptr()
    if one != 1 or (row | head) % unit or at % (2 * unit) or dim % 8 or not 0 < dim <= MAX_DIM or heads < 1:
        if dim < 1 or heads < 1 or dim % 8 or dim > MAX_DIM:
            raise ValueError("%s: dim must be a multiple of 8 up to %d, got %d" % (name, MAX_DIM, dim))
        raise ValueError("%s must be contiguous in its last dimension, its rows and heads on %d-byte boundaries"
                         % (name, 2 * unit))
    forward_only(x, name)
    return _native.AimgHeads(at, n, row, head, heads, dim)


def _refuse(x: torch.Tensor, name: str, dtype: torch.dtype, index: int) -> None:
    if x.get_device() < 0:
        raise RuntimeError("attention runs on the GPU only; got %s on %s" % (name, x.device))
    if x.dim() != 3 or x.dtype not in _TYPES:
        raise ValueError("%s must be a bf16 or fp16 [rows, heads, dim] tensor" % name)
    raise ValueError("%s must be %s on cuda:%d" % (name, dtype, index))


def _query(q: torch.Tensor) -> tuple[_native.AimgHeads, int, int]:
    """q's descriptor, its GPU and its type's number."""
    index, kind = q.get_device(), _TYPES.get(q.dtype)
    if kind is None or index < 0:
        _refuse(q, "q", q.dtype, index)
    return _heads(q, "q", q.dtype, index), index, kind


def _result(q: torch.Tensor, qd: _native.AimgHeads, out: torch.Tensor | None, index: int) -> tuple[torch.Tensor, _native.AimgHeads]:
    """The output tensor and its descriptor."""
    if out is None:
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
        return out, _native.AimgHeads(out.data_ptr(), qd.n_rows, qd.heads * qd.dim, qd.dim, qd.heads, qd.dim)
    if out.shape != q.shape:
        raise ValueError("out must have q's shape %s" % (tuple(q.shape),))
    return out, _heads(out, "out", q.dtype, index, unit=4)


def _offsets(x: torch.Tensor, name: str, index: int) -> int:
    if x.dtype is not torch.int32 or x.dim() != 1 or x.get_device() != index or not x.is_contiguous():
        raise ValueError("%s must be a contiguous 1-D int32 tensor on cuda:%d" % (name, index))
    return x.data_ptr()


def _scale(scale: float | None, dim: int) -> float:
    scale = dim ** -0.5 if scale is None else float(scale)
    if not 0.0 < scale < math.inf:
        raise ValueError("scale must be a positive number, got %r" % scale)
    return scale


def _lse(lse: torch.Tensor | None, q: torch.Tensor) -> int | None:
    if lse is None:
        return None
    if lse.dtype is not torch.float32 or lse.device != q.device or lse.shape != q.shape[:2] or not lse.is_contiguous():
        raise ValueError("lse must be a contiguous fp32 [%d, %d] tensor on %s" % (*q.shape[:2], q.device))
    return lse.data_ptr()


def _workspace(nbytes: int, q: torch.Tensor) -> torch.Tensor | None:
    """Scratch memory from torch's allocator on the current stream, which the
    launches use. The caller holds the tensor until they are made: the entries
    release the interpreter's lock, and another thread on this stream would be
    given memory that no tensor holds, for work that runs before them."""
    return torch.empty(nbytes, dtype=torch.uint8, device=q.device) if nbytes else None


def launch(entry, index: int, *args) -> None:
    """entry(*args, stream) with GPU ``index`` current, on its current stream.
    (The handle itself: a torch.cuda.Stream object and a device context cost
    2 us of a call.)"""
    if _current_device() == index:
        status = entry(*args, _stream_handle(index))
    else:
        with torch.cuda.device(index):
            status = entry(*args, _stream_handle(index))
    if status:
        _native.check(status)


@functools.lru_cache(maxsize=1024)
def _prompt_workspace_nbytes(n: int, n_keys: int, heads: int, kv_heads: int, dim: int, n_seqs: int) -> int:
    nbytes = ctypes.c_size_t(0)
    _native.check(_native.lib().aimg_prompt_workspace_nbytes(n, n_keys, heads, kv_heads, dim, n_seqs, ctypes.byref(nbytes)))
    return nbytes.value


def prompt_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, q_offsets: torch.Tensor,
                     k_offsets: torch.Tensor | None = None, *, scale: float | None = None,
                     out: torch.Tensor | None = None, lse: torch.Tensor | None = None) -> torch.Tensor:
    """Causal attention of packed prompts, on the current stream.

    q: [rows, heads, dim]; k, v: [keys, kv_heads, dim] with heads a multiple of
    kv_heads (head h reads key/value head h // (heads / kv_heads)); bf16 or
    fp16, dim a multiple of 8 up to 256. Sequence b has rows q_offsets[b] ..
    q_offsets[b + 1] - 1 and keys k_offsets[b] .. k_offsets[b + 1] - 1 (int32
    tensors on the GPU; k_offsets is q_offsets when not given). Its last row sees all its
    keys, the row before it all but the last, and so on: a prompt that
    continues a context has more keys than rows, and a row that sees no key
    gives zeros. scale is 1 / sqrt(dim) when not given.

    Returns out (q's shape and type; rows of no sequence are not written).
    lse, fp32 [rows, heads], receives log(sum(exp(scale * q.k))) when given.
    Results do not vary between calls. No gradients: inputs that require one
    are refused outside torch.no_grad()."""
    qd, index, kind = _query(q)
    kd, vd = _heads(k, "k", q.dtype, index), _heads(v, "v", q.dtype, index)
    if kd.n_rows != vd.n_rows or kd.heads != vd.heads or kd.dim != qd.dim or vd.dim != qd.dim:
        raise ValueError("k and v must have one shape and q's dim, got %s, %s and %s"
                         % (tuple(k.shape), tuple(v.shape), tuple(q.shape)))
    if qd.heads % kd.heads:
        raise ValueError("q's %d heads must be a multiple of k's %d" % (qd.heads, kd.heads))
    q_at = _offsets(q_offsets, "q_offsets", index)
    n_seqs = q_offsets.shape[0] - 1
    if k_offsets is None:
        if qd.n_rows != kd.n_rows:
            raise ValueError("q has %d rows and k %d: k_offsets is needed" % (qd.n_rows, kd.n_rows))
        k_at, n_keys = q_at, n_seqs
    else:
        k_at, n_keys = _offsets(k_offsets, "k_offsets", index), k_offsets.shape[0] - 1
    if n_seqs < 0 or n_keys != n_seqs:
        raise ValueError("q_offsets and k_offsets must have one entry more than there are sequences, got %d and %d"
                         % (n_seqs + 1, n_keys + 1))
    out, od = _result(q, qd, out, index)
    nbytes = _prompt_workspace_nbytes(qd.n_rows, kd.n_rows, qd.heads, kd.heads, qd.dim, n_seqs)
    work = _workspace(nbytes, q)
    launch(_native.lib().aimg_prompt_attention, index, qd, kd, vd, od, q_at, k_at, n_seqs, kind, _scale(scale, qd.dim), _lse(lse, q),
           work.data_ptr() if nbytes else None, nbytes)
    return out


def describe_pages(k_pages: torch.Tensor, v_pages: torch.Tensor, page_table: torch.Tensor,
                   lengths: torch.Tensor) -> _native.AimgPages:
    """The descriptor of one layer's paged keys and values [n_pages, kv_heads,
    page_size, dim] (any strides with a contiguous last dimension and whole
    16-byte pieces, the same for both) and of the int32 page table [max_seqs,
    max_pages] and lengths [max_seqs]."""
    index = k_pages.get_device()
    if index < 0:
        raise RuntimeError("the cache lives on the GPU only; got k_pages on %s" % k_pages.device)
    if k_pages.dim() != 4 or k_pages.dtype not in _TYPES:
        raise ValueError("k_pages must be a bf16 or fp16 [n_pages, kv_heads, page_size, dim] tensor")
    shape, strides = k_pages.shape, k_pages.stride()
    if v_pages.shape != shape or v_pages.dtype is not k_pages.dtype or v_pages.stride() != strides or v_pages.get_device() != index:
        raise ValueError("v_pages must have k_pages' shape, type, strides and device")
    if page_table.dtype is not torch.int32 or page_table.dim() != 2 or page_table.get_device() != index or page_table.stride(1) != 1:
        raise ValueError("page_table must be an int32 [max_seqs, max_pages] tensor on cuda:%d, its rows contiguous" % index)
    max_seqs, max_pages = page_table.shape
    if lengths.dtype is not torch.int32 or lengths.dim() != 1 or lengths.shape[0] != max_seqs or lengths.get_device() != index \
            or not lengths.is_contiguous():
        raise ValueError("lengths must be a contiguous int32 [%d] tensor on cuda:%d" % (max_seqs, index))
    n_pages, kv_heads, page_size, dim = shape
    page, head, slot, one = strides
    k_at, v_at = k_pages.data_ptr(), v_pages.data_ptr()
    if one != 1 or (page | head | slot) % 8 or (k_at | v_at) % 16:
        raise ValueError("k_pages and v_pages must be contiguous in their last dimension, their rows on 16-byte boundaries")
    return _native.AimgPages(k_at, v_at, page_table.data_ptr(), lengths.data_ptr(), page, slot, head, page_table.stride(0), n_pages,
                             page_size, kv_heads, dim, max_seqs, max_pages)


@functools.lru_cache(maxsize=1024)
def _tree_workspace_nbytes(n: int, heads: int, kv_heads: int, dim: int, n_seqs: int, max_drafts: int, max_context: int) -> int:
    nbytes = ctypes.c_size_t(0)
    _native.check(_native.lib().aimg_tree_workspace_nbytes(n, heads, kv_heads, dim, n_seqs, max_drafts, max_context,
                                                           ctypes.byref(nbytes)))
    return nbytes.value


def tree_attention(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, page_table: torch.Tensor,
                   lengths: torch.Tensor, seqs: torch.Tensor, draft_offsets: torch.Tensor,
                   masks: torch.Tensor | None = None, *, max_drafts: int, max_context: int | None = None,
                   scale: float | None = None, out: torch.Tensor | None = None,
                   lse: torch.Tensor | None = None) -> torch.Tensor:
    """Attention of drafted tokens over a paged cache, on the current stream:
    the verification pass of drafted trees (afterimage/runtime/
    streaming_engine.py:2554-2556 runs step_k + 1 positions), and plain
    decoding with one token a sequence.

    q: [rows, heads, dim]. Rows draft_offsets[b] .. draft_offsets[b + 1] - 1
    (at most max_drafts) are the drafted tokens of cache slot seqs[b]; their
    keys and values are in the cache already, at positions lengths[slot] and
    after. k_pages, v_pages: one layer's pages [n_pages, kv_heads, page_size,
    dim]; page_table [max_seqs, max_pages] and lengths [max_seqs]: int32, on
    the GPU like seqs and draft_offsets.

    A token sees every position before lengths[slot], and drafted token j of
    its sequence where bit j % 64 of masks[row, j // 64] is set (int64,
    tree_masks makes them); without masks, the drafted tokens up to itself. A
    token that sees nothing gives zeros. max_context, the longest context to
    expect (all that the table can hold when not given), decides how the work is
    split, nothing else.

    Returns out (q's shape and type; rows of no sequence, or past its first
    max_drafts, are not written); lse as in prompt_attention. Results do not
    vary between calls. No gradients, as there."""
    qd, index, kind = _query(q)
    pages = describe_pages(k_pages, v_pages, page_table, lengths)
    forward_only(k_pages, "k_pages")
    forward_only(v_pages, "v_pages")
    if k_pages.dtype is not q.dtype or k_pages.get_device() != index:
        raise ValueError("k_pages must be %s on %s" % (q.dtype, q.device))
    heads, kv_heads, dim = qd.heads, pages.kv_heads, qd.dim
    if pages.dim != dim or heads % kv_heads:
        raise ValueError("q's dim %d must be the pages' %d, its %d heads a multiple of their %d"
                         % (dim, pages.dim, heads, kv_heads))
    seqs_at, at = _offsets(seqs, "seqs", index), _offsets(draft_offsets, "draft_offsets", index)
    n_seqs, n = seqs.shape[0], qd.n_rows
    if draft_offsets.shape[0] != n_seqs + 1:
        raise ValueError("draft_offsets must have one entry more than seqs, got %d and %d" % (draft_offsets.shape[0], n_seqs))
    if max_drafts < 1:
        raise ValueError("max_drafts must be at least 1, got %d" % max_drafts)
    masks_at, words = None, 0
    if masks is not None:
        if masks.dtype is not torch.int64 or masks.dim() != 2 or masks.shape[0] != n or masks.get_device() != index \
                or not masks.is_contiguous() or masks.shape[1] * 64 < max_drafts:
            raise ValueError("masks must be a contiguous int64 [%d, at least %d] tensor on cuda:%d"
                             % (n, -(-max_drafts // 64), index))
        masks_at, words = masks.data_ptr(), masks.shape[1]
    if max_context is None:
        max_context = pages.max_pages * pages.page_size
    elif max_context < 0:
        raise ValueError("max_context must not be negative, got %d" % max_context)
    out, od = _result(q, qd, out, index)
    nbytes = _tree_workspace_nbytes(n, heads, kv_heads, dim, n_seqs, max_drafts, max_context)
    work = _workspace(nbytes, q)
    launch(_native.lib().aimg_tree_attention, index, qd, pages, od, seqs_at, at, n_seqs, masks_at, words, max_drafts, max_context,
           kind, _scale(scale, dim), _lse(lse, q), work.data_ptr() if nbytes else None, nbytes)
    return out


def tree_masks(parents: torch.Tensor, draft_offsets: torch.Tensor, max_drafts: int) -> torch.Tensor:
    """The masks of tree_attention from each drafted token's parent: int32
    indices within the token's sequence, earlier than the token; any other
    number (-1) for a token that follows the context. A token sees itself
    and its ancestors. int64 [rows, ceil(max_drafts / 64)]."""
    index = parents.get_device()
    if index < 0:
        raise RuntimeError("attention runs on the GPU only; got parents on %s" % parents.device)
    at, up = _offsets(draft_offsets, "draft_offsets", index), _offsets(parents, "parents", index)
    if max_drafts < 1 or draft_offsets.shape[0] < 1:
        raise ValueError("max_drafts must be at least 1 and draft_offsets not empty")
    n, words = parents.shape[0], -(-max_drafts // 64)
    masks = torch.empty((n, words), dtype=torch.int64, device=parents.device)
    launch(_native.lib().aimg_tree_masks, index, up, at, draft_offsets.shape[0] - 1, n, words, masks.data_ptr())
    return masks
