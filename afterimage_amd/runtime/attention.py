"""Attention between a decoder layer's projections: whole prompts, and drafted
tokens over a paged cache.

The reference leaves attention to the model's own forward pass
(afterimage/runtime/streaming_engine.py:2154-2213 drives it); these are the
products a program runs between the q/k/v projections whose weights it decodes
and the output projection. Elements are bf16 or fp16; scores, softmax
statistics and sums are fp32. Work is ordered on the current stream and nothing
here synchronises.
"""
from __future__ import annotations

import ctypes
import functools
import math

import torch

from .. import _native

MAX_DIM = 256

_TYPES = {torch.bfloat16: _native.AIMG_BF16, torch.float16: _native.AIMG_FP16}


def _heads(x: torch.Tensor, name: str, like: torch.Tensor | None = None, written: bool = False) -> _native.AimgHeads:
    """The descriptor of rows of heads [n, heads, dim], any row and head
    strides that keep whole 16-byte pieces aligned (8 where written)."""
    if x.device.type != "cuda":
        raise RuntimeError("attention runs on the GPU only; got %s on %s" % (name, x.device))
    if x.dim() != 3 or x.dtype not in _TYPES:
        raise ValueError("%s must be a bf16 or fp16 [rows, heads, dim] tensor" % name)
    if like is not None and (x.dtype != like.dtype or x.device != like.device):
        raise ValueError("%s must be %s on %s" % (name, like.dtype, like.device))
    n, heads, dim = x.shape
    row, head, one = x.stride()
    if dim < 1 or heads < 1 or dim % 8 or dim > MAX_DIM:
        raise ValueError("%s: dim must be a multiple of 8 up to %d, got %d" % (name, MAX_DIM, dim))
    unit = 4 if written else 8
    if one != 1 or row % unit or head % unit or x.data_ptr() % (2 * unit):
        raise ValueError("%s must be contiguous in its last dimension, its rows and heads on %d-byte boundaries"
                         % (name, 2 * unit))
    return _native.AimgHeads(x.data_ptr(), n, row, head, heads, dim)


def _offsets(x: torch.Tensor, name: str, device) -> int:
    if x.dtype != torch.int32 or x.dim() != 1 or x.device != device or not x.is_contiguous():
        raise ValueError("%s must be a contiguous 1-D int32 tensor on %s" % (name, device))
    return x.data_ptr()


def _scale(scale: float | None, dim: int) -> float:
    scale = dim ** -0.5 if scale is None else float(scale)
    if not 0.0 < scale < math.inf:
        raise ValueError("scale must be a positive number, got %r" % scale)
    return scale


def _lse(lse: torch.Tensor | None, q: torch.Tensor) -> int | None:
    if lse is None:
        return None
    if lse.dtype != torch.float32 or lse.device != q.device or lse.shape != q.shape[:2] or not lse.is_contiguous():
        raise ValueError("lse must be a contiguous fp32 [%d, %d] tensor on %s" % (*q.shape[:2], q.device))
    return lse.data_ptr()


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
    lse, fp32 [rows, heads], receives log(sum(exp(scale * q.k))) when given."""
    qd = _heads(q, "q")
    kd, vd = _heads(k, "k", q), _heads(v, "v", q)
    dev = q.device
    if k.shape != v.shape or k.shape[2] != q.shape[2]:
        raise ValueError("k and v must have one shape and q's dim, got %s, %s and %s"
                         % (tuple(k.shape), tuple(v.shape), tuple(q.shape)))
    if q.shape[1] % k.shape[1]:
        raise ValueError("q's %d heads must be a multiple of k's %d" % (q.shape[1], k.shape[1]))
    q_at = _offsets(q_offsets, "q_offsets", dev)
    if k_offsets is None:
        if q.shape[0] != k.shape[0]:
            raise ValueError("q has %d rows and k %d: k_offsets is needed" % (q.shape[0], k.shape[0]))
        k_offsets, k_at = q_offsets, q_at
    else:
        k_at = _offsets(k_offsets, "k_offsets", dev)
    n_seqs = q_offsets.shape[0] - 1
    if n_seqs < 0 or k_offsets.shape[0] != n_seqs + 1:
        raise ValueError("q_offsets and k_offsets must have one entry more than there are sequences, got %d and %d"
                         % (q_offsets.shape[0], k_offsets.shape[0]))
    scale = _scale(scale, q.shape[2])
    if out is None:
        out = torch.empty(q.shape, dtype=q.dtype, device=dev)
    elif out.shape != q.shape:
        raise ValueError("out must have q's shape %s" % (tuple(q.shape),))
    od = _heads(out, "out", q, written=True)
    lse_at = _lse(lse, q)
    with torch.cuda.device(dev):
        _native.check(_native.lib().aimg_prompt_attention(
            ctypes.byref(qd), ctypes.byref(kd), ctypes.byref(vd), ctypes.byref(od), q_at, k_at, n_seqs,
            _TYPES[q.dtype], scale, lse_at, torch.cuda.current_stream(dev).cuda_stream))
    return out


def describe_pages(k_pages: torch.Tensor, v_pages: torch.Tensor, page_table: torch.Tensor,
                   lengths: torch.Tensor) -> _native.AimgPages:
    """The descriptor of one layer's paged keys and values [n_pages, kv_heads,
    page_size, dim] (any strides with a contiguous last dimension and whole
    16-byte pieces, the same for both) and of the int32 page table [max_seqs,
    max_pages] and lengths [max_seqs]."""
    dev = k_pages.device
    if dev.type != "cuda":
        raise RuntimeError("the cache lives on the GPU only; got k_pages on %s" % dev)
    if k_pages.dim() != 4 or k_pages.dtype not in _TYPES:
        raise ValueError("k_pages must be a bf16 or fp16 [n_pages, kv_heads, page_size, dim] tensor")
    if v_pages.shape != k_pages.shape or v_pages.dtype != k_pages.dtype or v_pages.stride() != k_pages.stride() \
            or v_pages.device != dev:
        raise ValueError("v_pages must have k_pages' shape, type, strides and device")
    if page_table.dtype != torch.int32 or page_table.dim() != 2 or page_table.device != dev or page_table.stride(1) != 1:
        raise ValueError("page_table must be an int32 [max_seqs, max_pages] tensor on %s, its rows contiguous" % dev)
    if lengths.dtype != torch.int32 or lengths.shape != page_table.shape[:1] or lengths.device != dev \
            or not lengths.is_contiguous():
        raise ValueError("lengths must be a contiguous int32 [%d] tensor on %s" % (page_table.shape[0], dev))
    n_pages, kv_heads, page_size, dim = k_pages.shape
    page, head, slot, one = k_pages.stride()
    if one != 1 or page % 8 or head % 8 or slot % 8 or (k_pages.data_ptr() | v_pages.data_ptr()) % 16:
        raise ValueError("k_pages and v_pages must be contiguous in their last dimension, their rows on 16-byte boundaries")
    return _native.AimgPages(k_pages.data_ptr(), v_pages.data_ptr(), page_table.data_ptr(), lengths.data_ptr(), page, slot, head,
                             page_table.stride(0), n_pages, page_size, kv_heads, dim, page_table.shape[0], page_table.shape[1])


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

    Returns out (q's shape and type); lse as in prompt_attention. Results do
    not vary between calls."""
    qd = _heads(q, "q")
    dev = q.device
    pages = describe_pages(k_pages, v_pages, page_table, lengths)
    if k_pages.dtype != q.dtype or k_pages.device != dev:
        raise ValueError("k_pages must be %s on %s" % (q.dtype, dev))
    if pages.dim != qd.dim or qd.heads % pages.kv_heads:
        raise ValueError("q's dim %d must be the pages' %d, its %d heads a multiple of their %d"
                         % (qd.dim, pages.dim, qd.heads, pages.kv_heads))
    n_seqs = seqs.shape[0]
    seqs_at, at = _offsets(seqs, "seqs", dev), _offsets(draft_offsets, "draft_offsets", dev)
    if draft_offsets.shape[0] != n_seqs + 1:
        raise ValueError("draft_offsets must have one entry more than seqs, got %d and %d" % (draft_offsets.shape[0], n_seqs))
    if max_drafts < 1:
        raise ValueError("max_drafts must be at least 1, got %d" % max_drafts)
    masks_at, words = None, 0
    if masks is not None:
        if masks.dtype != torch.int64 or masks.dim() != 2 or masks.shape[0] != qd.n_rows or masks.device != dev \
                or not masks.is_contiguous() or masks.shape[1] * 64 < max_drafts:
            raise ValueError("masks must be a contiguous int64 [%d, at least %d] tensor on %s"
                             % (qd.n_rows, -(-max_drafts // 64), dev))
        masks_at, words = masks.data_ptr(), masks.shape[1]
    if max_context is None:
        max_context = pages.max_pages * pages.page_size
    elif max_context < 0:
        raise ValueError("max_context must not be negative, got %d" % max_context)
    scale = _scale(scale, qd.dim)
    if out is None:
        out = torch.empty(q.shape, dtype=q.dtype, device=dev)
    elif out.shape != q.shape:
        raise ValueError("out must have q's shape %s" % (tuple(q.shape),))
    od = _heads(out, "out", q, written=True)
    lse_at = _lse(lse, q)
    nbytes = _tree_workspace_nbytes(qd.n_rows, qd.heads, pages.kv_heads, qd.dim, n_seqs, max_drafts, max_context)
    with torch.cuda.device(dev):
        work = torch.empty(nbytes, dtype=torch.uint8, device=dev) if nbytes else None
        _native.check(_native.lib().aimg_tree_attention(
            ctypes.byref(qd), ctypes.byref(pages), ctypes.byref(od), seqs_at, at, n_seqs, masks_at, words, max_drafts,
            max_context, _TYPES[q.dtype], scale, lse_at, work.data_ptr() if nbytes else None, nbytes,
            torch.cuda.current_stream(dev).cuda_stream))
    return out


def tree_masks(parents: torch.Tensor, draft_offsets: torch.Tensor, max_drafts: int) -> torch.Tensor:
    """The masks of tree_attention from each drafted token's parent: int32
    indices within the token's sequence, earlier than the token; any other
    number (-1) for a token that follows the context. A token sees itself
    and its ancestors. int64 [rows, ceil(max_drafts / 64)]."""
    dev = parents.device
    if dev.type != "cuda":
        raise RuntimeError("attention runs on the GPU only; got parents on %s" % dev)
    at, up = _offsets(draft_offsets, "draft_offsets", dev), _offsets(parents, "parents", dev)
    if max_drafts < 1 or draft_offsets.shape[0] < 1:
        raise ValueError("max_drafts must be at least 1 and draft_offsets not empty")
    n, words = parents.shape[0], -(-max_drafts // 64)
    masks = torch.empty((n, words), dtype=torch.int64, device=dev)
    with torch.cuda.device(dev):
        _native.check(_native.lib().aimg_tree_masks(up, at, draft_offsets.shape[0] - 1, n, words, masks.data_ptr(),
                                                    torch.cuda.current_stream(dev).cuda_stream))
    return masks
