"""A paged key/value cache whose page table lives on the GPU.

The reference keeps a model's cache in the model's own forward pass and reserves
bytes for it (afterimage/runtime/config.py:127-140); a program that verifies
drafted tokens against decoded weights needs its steps: append a layer's rows,
attend over them (attention.tree_attention), keep a tree's accepted path, branch
and drop sequences. Every step runs on the GPU, ordered on the current stream,
from device tensors: none waits for the host. What a step cannot do (no free
pages, a slot that does not exist) it leaves undone and records in ``status``;
``check`` reads it.

A sequence is a slot. Slot s holds the pages page_table[s, :held[s]] for its
lengths[s] positions and those to come; position j is row j % page_size of page
page_table[s, j // page_size], the same page in every layer, for keys and for
values. refs[p] slots hold page p. Free pages are given out lowest first, in the
order of a call. A call names a slot once.
"""
from __future__ import annotations

import ctypes

import torch

from .. import _native
from .attention import forward_only, launch, tree_attention

MAX_SEQS = 8192      # sequences of one call
MAX_PAGES = (1 << 20) - 1

_PROBLEMS = ((1, "too few free pages"), (2, "positions past a sequence's pages or its row of the page table"),
             (4, "a slot, page, source or number of rows that does not exist"))


def _int32(x: torch.Tensor, name: str, shape: tuple, index: int) -> int:
    if x.dtype is not torch.int32 or x.get_device() != index or x.shape != shape or not x.is_contiguous():
        raise ValueError("%s must be a contiguous int32 %s tensor on cuda:%d" % (name, list(shape), index))
    return x.data_ptr()


class PagedKVCache:
    """Pages of keys and values for every layer of a model, over tensors on one GPU:

    pool        [n_layers, 2, n_pages, kv_heads, page_size, dim], bf16 or fp16
    page_table  int32 [max_seqs, max_pages], -1 where a slot holds no page
    lengths     int32 [max_seqs], positions of each slot
    held        int32 [max_seqs], pages of each slot
    refs        int32 [n_pages], slots that hold each page
    status      int32 [1], what went wrong (see check)

    ``allocate`` makes an empty one. The tensors are used in place and are the
    cache's whole state. ``seqs``, ``src`` and ``dst`` below are slots: int32
    tensors on the GPU of at most 8192 entries."""

    def __init__(self, pool: torch.Tensor, page_table: torch.Tensor, lengths: torch.Tensor, held: torch.Tensor,
                 refs: torch.Tensor, status: torch.Tensor):
        index = pool.get_device()
        if index < 0:
            raise RuntimeError("the cache lives on the GPU only; got the pool on %s" % pool.device)
        if pool.dim() != 6 or pool.shape[1] != 2 or pool.dtype not in (torch.bfloat16, torch.float16) \
                or not pool.is_contiguous() or pool.numel() == 0:
            raise ValueError("pool must be a contiguous bf16 or fp16 [n_layers, 2, n_pages, kv_heads, page_size, dim] tensor")
        if page_table.dim() != 2 or page_table.numel() == 0:
            raise ValueError("page_table must be a contiguous int32 [max_seqs, max_pages] tensor on cuda:%d" % index)
        self.n_layers, _, self.n_pages, self.kv_heads, self.page_size, self.dim = pool.shape
        self.max_seqs, self.max_pages = page_table.shape
        if self.dim % 8 or pool.data_ptr() % 16:
            raise ValueError("pool: dim must be a multiple of 8 and its memory 16-byte aligned")
        if self.n_pages > MAX_PAGES or self.max_pages * self.page_size >= 1 << 30:
            raise ValueError("pool: at most %d pages, and fewer than 2^30 positions a sequence" % MAX_PAGES)
        self._cache = _native.AimgCache(
            pool.data_ptr(), _int32(page_table, "page_table", (self.max_seqs, self.max_pages), index),
            _int32(lengths, "lengths", (self.max_seqs,), index), _int32(held, "held", (self.max_seqs,), index),
            _int32(refs, "refs", (self.n_pages,), index), _int32(status, "status", (1,), index),
            self.n_layers, self.n_pages, self.kv_heads, self.page_size, self.dim, self.max_seqs, self.max_pages)
        self.device = pool.device
        self._index = index
        self._lib = _native.lib()
        self.pool, self.page_table, self.lengths, self.held, self.refs, self.status = \
            pool, page_table, lengths, held, refs, status
        nbytes = ctypes.c_size_t(0)
        _native.check(self._lib.aimg_cache_compact_workspace_nbytes(self._cache, ctypes.byref(nbytes)))
        # Scratch memory of compact, of one size and so kept as long as the cache: calls change one cache and run in order.
        self._compact_work = torch.empty(nbytes.value, dtype=torch.uint8, device=self.device)
        self._used = torch.empty((), dtype=torch.int32, device=self.device)

    @classmethod
    def allocate(cls, n_layers: int, n_pages: int, page_size: int, kv_heads: int, dim: int, max_seqs: int, max_pages: int,
                 dtype: torch.dtype = torch.bfloat16, device="cuda") -> "PagedKVCache":
        """An empty cache. The pool's memory is not cleared."""
        def ints(*shape, value=0):
            return torch.full(shape, value, dtype=torch.int32, device=device)
        pool = torch.empty((n_layers, 2, n_pages, kv_heads, page_size, dim), dtype=dtype, device=device)
        return cls(pool, ints(max_seqs, max_pages, value=-1), ints(max_seqs), ints(max_seqs), ints(n_pages), ints(1))

    def _seqs(self, x: torch.Tensor, name: str = "seqs") -> tuple[int, int]:
        """The address and the number of a call's slots."""
        if x.dtype is not torch.int32 or x.dim() != 1 or x.get_device() != self._index or not x.is_contiguous():
            raise ValueError("%s must be a contiguous 1-D int32 tensor on cuda:%d" % (name, self._index))
        n = x.shape[0]
        if n > MAX_SEQS:
            raise ValueError("%s: at most %d slots a call, got %d" % (name, MAX_SEQS, n))
        return x.data_ptr(), n

    def keys(self, layer: int) -> torch.Tensor:
        """One layer's key pages [n_pages, kv_heads, page_size, dim]."""
        return self.pool[layer, 0]

    def values(self, layer: int) -> torch.Tensor:
        return self.pool[layer, 1]

    def reserve(self, seqs: torch.Tensor, tokens: torch.Tensor) -> None:
        """Pages for tokens[b] (int32) positions past slot seqs[b]'s length,
        for all slots or for none."""
        at, n = self._seqs(seqs)
        launch(self._lib.aimg_cache_reserve, self._index, self._cache, at, _int32(tokens, "tokens", (n,), self._index), n)

    def _rows(self, x: torch.Tensor, name: str) -> _native.AimgHeads:
        if x.dim() != 3 or x.dtype is not self.pool.dtype or x.get_device() != self._index \
                or x.shape[1:] != (self.kv_heads, self.dim):
            raise ValueError("%s must be a %s [rows, %d, %d] tensor on %s"
                             % (name, self.pool.dtype, self.kv_heads, self.dim, self.device))
        row, head, one = x.stride()
        if one != 1 or (row | head) % 8 or x.data_ptr() % 16:
            raise ValueError("%s must be contiguous in its last dimension, its rows and heads on 16-byte boundaries" % name)
        forward_only(x, name)
        return _native.AimgHeads(x.data_ptr(), x.shape[0], row, head, x.shape[1], x.shape[2])

    def append(self, layer: int, k: torch.Tensor, v: torch.Tensor, seqs: torch.Tensor, offsets: torch.Tensor) -> None:
        """Rows offsets[b] .. offsets[b + 1] - 1 of k and v [rows, kv_heads,
        dim] into slot seqs[b]'s reserved pages, from its length on; lengths
        stay (advance or commit moves them, once every layer has its rows)."""
        kd, vd = self._rows(k, "k"), self._rows(v, "v")
        if not 0 <= layer < self.n_layers:
            raise ValueError("layer must be in 0..%d, got %d" % (self.n_layers - 1, layer))
        if k.shape != v.shape:
            raise ValueError("k and v must have one shape, got %s and %s" % (tuple(k.shape), tuple(v.shape)))
        at, n = self._seqs(seqs)
        launch(self._lib.aimg_cache_append, self._index, self._cache, layer, kd, vd, at,
               _int32(offsets, "offsets", (n + 1,), self._index), n)

    def advance(self, seqs: torch.Tensor, offsets: torch.Tensor) -> None:
        """Slot seqs[b]'s length grows by offsets[b + 1] - offsets[b], the rows that were appended."""
        at, n = self._seqs(seqs)
        launch(self._lib.aimg_cache_advance, self._index, self._cache, at, _int32(offsets, "offsets", (n + 1,), self._index), n)

    def attend(self, layer: int, q: torch.Tensor, seqs: torch.Tensor, draft_offsets: torch.Tensor,
               masks: torch.Tensor | None = None, **options) -> torch.Tensor:
        """tree_attention of q over one layer of this cache."""
        return tree_attention(q, self.keys(layer), self.values(layer), self.page_table, self.lengths, seqs, draft_offsets,
                              masks, **options)

    def commit(self, seqs: torch.Tensor, accepted: torch.Tensor, counts: torch.Tensor,
               new_lengths: torch.Tensor | None = None) -> torch.Tensor:
        """Keeps counts[b] drafted tokens of slot seqs[b], those of indices
        accepted[b, :counts[b]] (int32, rising: a path of the tree): in every
        layer their rows move to the positions from the length on, and the
        length grows by counts[b] (0 to accepted's width; anything else is left
        undone and recorded). The new lengths go to new_lengths (int32
        [max_seqs], the call's slots only) where given, in place otherwise.
        Returns the lengths written."""
        at, n = self._seqs(seqs)
        if accepted.dim() != 2:
            raise ValueError("accepted must be a contiguous int32 [%d, most] tensor on %s" % (n, self.device))
        most = accepted.shape[1]
        lengths = self.lengths if new_lengths is None else new_lengths
        launch(self._lib.aimg_cache_commit, self._index, self._cache, at, _int32(accepted, "accepted", (n, most), self._index), most,
               _int32(counts, "counts", (n,), self._index), n, _int32(lengths, "new_lengths", (self.max_seqs,), self._index))
        return lengths

    def fork(self, src: torch.Tensor, dst: torch.Tensor) -> None:
        """Slot dst[i] becomes a branch of slot src[i], all pairs at once (a
        source may itself be replaced, as when beams are reordered; a pair of
        one slot stays). Branches share the source's full pages; the rows of its
        last page are copied to a free one. What a slot held before is given
        back after the copies."""
        s, n = self._seqs(src, "src")
        d = _int32(dst, "dst", (n,), self._index)
        nbytes = 4 * n * (2 + self.max_pages)
        # The call's own, from torch's allocator on the current stream: a buffer
        # kept here would have to grow, and a captured graph or another stream
        # may still use the smaller one.
        work = torch.empty(nbytes, dtype=torch.uint8, device=self.device)
        launch(self._lib.aimg_cache_fork, self._index, self._cache, s, d, n, work.data_ptr(), nbytes)

    def release(self, seqs: torch.Tensor) -> None:
        """Empties the slots; pages that no other slot holds are free."""
        at, n = self._seqs(seqs)
        launch(self._lib.aimg_cache_release, self._index, self._cache, at, n)

    def compact(self, new_table: torch.Tensor | None = None, new_refs: torch.Tensor | None = None) -> torch.Tensor:
        """Moves the pages in use to the front of the pool, in every layer,
        with the fewest moves, and returns their number (int32, on the GPU).
        The page table and reference counts after the moves go to new_table and
        new_refs where given, in place otherwise."""
        table = self.page_table if new_table is None else new_table
        refs = self.refs if new_refs is None else new_refs
        used = torch.empty_like(self._used)
        launch(self._lib.aimg_cache_compact, self._index, self._cache,
               _int32(table, "new_table", (self.max_seqs, self.max_pages), self._index),
               _int32(refs, "new_refs", (self.n_pages,), self._index), used.data_ptr(), self._compact_work.data_ptr(),
               self._compact_work.shape[0])
        return used

    def check(self) -> None:
        """Waits for the work so far, raises RuntimeError where a step could
        not be done, and clears the status."""
        status = int(self.status.item())
        if status:
            self.status.zero_()
            raise RuntimeError("the cache: " + "; ".join(text for bit, text in _PROBLEMS if status & bit))
