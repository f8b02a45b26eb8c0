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

A cache may hold its elements in 8 bits (torch.float8_e4m3fn), half the bytes
that attention reads: a scale for each 16 positions of a page and head, keys and
values apart, says what they stand for (value * scale). Scales are powers of
two, the smallest that bring the largest of the 16 positions' elements to at
most 448. Rows are rounded to nearest as they come in; where later rows raise
the scale of their 16 positions, earlier elements below 2^-6 of it are rounded
again, by at most 2^-10 of it. Drafted rows are such rows, and what they round
stays rounded where they are rejected: what a sequence holds in 8 bits depends,
by that much, on what was drafted. Infinities become NaN.
"""
from __future__ import annotations

import ctypes

import torch

from .. import _native
from .attention import _TYPES, _query, attend, describe_pages, forward_only, launch

MAX_SEQS = 8192      # sequences of one call
MAX_PAGES = (1 << 20) - 1
BLOCK = 16           # positions that share a scale, in 8 bits
MAX_DIM = 256        # of a cache in 8 bits, and of rows that are turned or read

_PROBLEMS = ((1, "too few free pages"), (2, "positions past a sequence's pages or its row of the page table"),
             (4, "a slot, page, source or number of rows that does not exist"))


# What steps use of the cache's state is handed on by address.
_TENSORS = frozenset(("pool", "page_table", "lengths", "held", "refs", "status", "scales"))


def _int32(x: torch.Tensor, name: str, shape: tuple, index: int) -> int:
    if x.dtype is not torch.int32 or x.get_device() != index or x.shape != shape or not x.is_contiguous():
        raise ValueError("%s must be a contiguous int32 %s tensor on cuda:%d" % (name, list(shape), index))
    return x.data_ptr()


class PagedKVCache:
    """Pages of keys and values for every layer of a model, over tensors on one GPU:

    pool        [n_layers, 2, n_pages, kv_heads, page_size, dim], bf16, fp16 or
                float8_e4m3fn (dim and page_size then multiples of 16)
    page_table  int32 [max_seqs, max_pages], -1 where a slot holds no page
    lengths     int32 [max_seqs], positions of each slot
    held        int32 [max_seqs], pages of each slot
    refs        int32 [n_pages], slots that hold each page
    status      int32 [1], what went wrong (see check)
    scales      fp32 [n_layers, 2, n_pages, kv_heads, page_size / 16], of a pool
                in 8 bits alone

    ``allocate`` makes an empty one. The tensors are used in place and are the
    cache's whole state. Another tensor of the same shape and type may be put
    in an attribute's place: every step uses it from then on (captured graphs
    go on with the one they were captured with). ``seqs``, ``src`` and ``dst``
    below are slots: int32 tensors on the GPU of at most 8192 entries."""

    scales: torch.Tensor | None = None

    def __init__(self, pool: torch.Tensor, page_table: torch.Tensor, lengths: torch.Tensor, held: torch.Tensor,
                 refs: torch.Tensor, status: torch.Tensor, scales: torch.Tensor | None = None):
        index = pool.get_device()
        if index < 0:
            raise RuntimeError("the cache lives on the GPU only; got the pool on %s" % pool.device)
        if pool.dim() != 6 or pool.shape[1] != 2 or pool.dtype not in (torch.bfloat16, torch.float16, torch.float8_e4m3fn) \
                or not pool.is_contiguous() or pool.numel() == 0:
            raise ValueError("pool must be a contiguous bf16, fp16 or float8_e4m3fn [n_layers, 2, n_pages, kv_heads, page_size, dim] tensor")
        if page_table.dim() != 2 or page_table.numel() == 0:
            raise ValueError("page_table must be a contiguous int32 [max_seqs, max_pages] tensor on cuda:%d" % index)
        self.n_layers, _, self.n_pages, self.kv_heads, self.page_size, self.dim = pool.shape
        self.max_seqs, self.max_pages = page_table.shape
        if self.dim % 8 or pool.data_ptr() % 16:
            raise ValueError("pool: dim must be a multiple of 8 and its memory 16-byte aligned")
        if self.n_pages > MAX_PAGES or self.max_pages * self.page_size >= 1 << 30:
            raise ValueError("pool: at most %d pages, and fewer than 2^30 positions a sequence" % MAX_PAGES)
        self._scales_at = None
        if pool.dtype is torch.float8_e4m3fn:
            if self.dim % 16 or self.dim > MAX_DIM or self.page_size % BLOCK:
                raise ValueError("pool: in 8 bits dim must be a multiple of 16 up to %d and page_size one of %d" % (MAX_DIM, BLOCK))
            shape = (self.n_layers, 2, self.n_pages, self.kv_heads, self.page_size // BLOCK)
            if scales is None or scales.dtype is not torch.float32 or scales.get_device() != index or scales.shape != shape \
                    or not scales.is_contiguous():
                raise ValueError("scales must be a contiguous fp32 %s tensor on cuda:%d" % (list(shape), index))
            self._scales_at = scales.data_ptr()
        elif scales is not None:
            raise ValueError("scales belong to a pool of float8_e4m3fn")
        self.pool, self.page_table, self.lengths, self.held, self.refs, self.status, self.scales = \
            pool, page_table, lengths, held, refs, status, scales
        self._cache = _native.AimgCache(
            pool.data_ptr(), _int32(page_table, "page_table", (self.max_seqs, self.max_pages), index),
            _int32(lengths, "lengths", (self.max_seqs,), index), _int32(held, "held", (self.max_seqs,), index),
            _int32(refs, "refs", (self.n_pages,), index), _int32(status, "status", (1,), index),
            self.n_layers, self.n_pages, self.kv_heads, self.page_size, self.dim, self.max_seqs, self.max_pages)
        self.device = pool.device
        self._index = index
        # What attention is told of each layer. (Views of the tensors, and their checks, took 12 us of a call.)
        self._described = []
        for layer in range(self.n_layers):
            pages = describe_pages(pool[layer, 0], pool[layer, 1], page_table, lengths)
            at = None if scales is None else scales[layer]
            self._described.append((pages, None if scales is None else _native.AimgPageScales(
                at[0].data_ptr(), at[1].data_ptr(), at.stride(1), at.stride(2))))
        self._lib = _native.lib()
        nbytes = ctypes.c_size_t(0)
        _native.check(self._lib.aimg_cache_compact_workspace_nbytes(self._cache, ctypes.byref(nbytes)))
        # Scratch memory of compact, of one size and so kept as long as the cache: calls change one cache and run in order.
        self._compact_work = torch.empty(nbytes.value, dtype=torch.uint8, device=self.device)
        self._used = torch.empty((), dtype=torch.int32, device=self.device)

    def __setattr__(self, name: str, value) -> None:
        if name in _TENSORS and "_described" in self.__dict__:
            self._replace(name, value)
        object.__setattr__(self, name, value)

    def _replace(self, name: str, x) -> None:
        """Checks a tensor that takes an attribute's place, and moves the addresses that the steps hand on to it."""
        old = self.__dict__[name]
        if old is None or not isinstance(x, torch.Tensor) or x.shape != old.shape or x.dtype is not old.dtype or x.get_device() != self._index \
                or not x.is_contiguous() or x.data_ptr() % (16 if name == "pool" else 4):
            raise ValueError("%s must %s" % (name, "stay None: the pool has 16 bits" if old is None else "stay a contiguous %s %s tensor on %s%s" % (
                old.dtype, list(old.shape), self.device, ", its memory 16-byte aligned" if name == "pool" else "")))
        at = x.data_ptr()
        # (Descriptors of this cache's own: a copy of the object shares the ones it was copied with.)
        if name == "scales":
            self._scales_at = at
        else:
            self._cache = _native.AimgCache.from_buffer_copy(self._cache)
            setattr(self._cache, name, at)
        if name in ("held", "refs", "status"):
            return
        described = [(_native.AimgPages.from_buffer_copy(pages), None if scales is None else _native.AimgPageScales.from_buffer_copy(scales))
                     for pages, scales in self._described]
        for layer, (pages, scales) in enumerate(described):
            if name in ("page_table", "lengths"):
                setattr(pages, name, at)
            else:
                one = pages if name == "pool" else scales
                one.k = at + layer * x.stride(0) * x.element_size()
                one.v = one.k + x.stride(1) * x.element_size()
        self._described = described

    @classmethod
    def allocate(cls, n_layers: int, n_pages: int, page_size: int, kv_heads: int, dim: int, max_seqs: int, max_pages: int,
                 dtype: torch.dtype = torch.bfloat16, device="cuda") -> "PagedKVCache":
        """An empty cache, of bf16, fp16 or float8_e4m3fn elements. The pool's memory is not cleared."""
        def ints(*shape, value=0):
            return torch.full(shape, value, dtype=torch.int32, device=device)
        pool = torch.empty((n_layers, 2, n_pages, kv_heads, page_size, dim), dtype=dtype, device=device)
        scales = torch.empty((n_layers, 2, n_pages, kv_heads, page_size // BLOCK), dtype=torch.float32, device=device) \
            if dtype is torch.float8_e4m3fn else None
        return cls(pool, ints(max_seqs, max_pages, value=-1), ints(max_seqs), ints(max_seqs), ints(n_pages), ints(1), scales)

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

    def _heads(self, x: torch.Tensor, name: str, dtype: torch.dtype, heads: int) -> _native.AimgHeads:
        shape = x.shape
        if len(shape) != 3 or x.dtype is not dtype or x.get_device() != self._index or shape[1] != heads or shape[2] != self.dim:
            raise ValueError("%s must be a %s [rows, %d, %d] tensor on %s" % (name, dtype, heads, self.dim, self.device))
        row, head, one = x.stride()
        at = x.data_ptr()
        if one != 1 or (row | head) % 8 or at % 16:
            raise ValueError("%s must be contiguous in its last dimension, its rows and heads on 16-byte boundaries" % name)
        forward_only(x, name)
        return _native.AimgHeads(at, shape[0], row, head, heads, self.dim)

    def _rows(self, x: torch.Tensor, name: str) -> _native.AimgHeads:
        return self._heads(x, name, self.pool.dtype, self.kv_heads)

    def _type(self, x: torch.Tensor, name: str) -> int:
        """The number of the type of a call's rows: the pool's, or bf16 or fp16 for a pool in 8 bits."""
        kind = _TYPES.get(x.dtype)
        if kind is None or (self.scales is None and x.dtype is not self.pool.dtype):
            raise ValueError("%s must be %s, got %s" % (name, self.pool.dtype if self.scales is None else "bf16 or fp16", x.dtype))
        return kind

    def _layer(self, layer: int) -> int:
        if not 0 <= layer < self.n_layers:
            raise ValueError("layer must be in 0..%d, got %d" % (self.n_layers - 1, layer))
        return layer

    def append(self, layer: int, k: torch.Tensor, v: torch.Tensor, seqs: torch.Tensor, offsets: torch.Tensor) -> None:
        """Rows offsets[b] .. offsets[b + 1] - 1 of k and v [rows, kv_heads,
        dim] into slot seqs[b]'s reserved pages, from its length on; lengths
        stay (advance or commit moves them, once every layer has its rows). k
        and v have the pool's type, bf16 or fp16 for one in 8 bits."""
        if self.scales is not None:
            kind = self._type(k, "k")
            kd, vd = self._heads(k, "k", k.dtype, self.kv_heads), self._heads(v, "v", k.dtype, self.kv_heads)
        else:
            kd, vd = self._rows(k, "k"), self._rows(v, "v")
        self._layer(layer)
        if k.shape != v.shape:
            raise ValueError("k and v must have one shape, got %s and %s" % (tuple(k.shape), tuple(v.shape)))
        at, n = self._seqs(seqs)
        offsets_at = _int32(offsets, "offsets", (n + 1,), self._index)
        if self.scales is not None:
            launch(self._lib.aimg_cache_append_rotated, self._index, self._cache, self._scales_at, layer, None, kd, vd, None, at,
                   offsets_at, n, None, None, kind)
        else:
            launch(self._lib.aimg_cache_append, self._index, self._cache, layer, kd, vd, at, offsets_at, n)

    def append_rotated(self, layer: int, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, seqs: torch.Tensor,
                       offsets: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor, positions: torch.Tensor | None = None, *,
                       interleaved: bool = False, out: torch.Tensor | None = None) -> torch.Tensor:
        """append, with the rotation of q [rows, heads, dim] and k by their
        positions on the way; returns the turned q (out where given, which may
        be q itself but must not overlap it or k and v otherwise).

        cos and sin: fp32 [positions, half], contiguous, half at most dim / 2
        (attention.rotary_tables makes them): elements i and i + half of a row
        at position p turn by the angle of cos[p, i] and sin[p, i], or elements
        2 i and 2 i + 1 where interleaved; those from 2 half on stay. Row r's
        position is positions[r] (int32 [rows]; a drafted token's is that of
        its place in the tree), its place in the cache where not given. Rows
        that are turned are rounded once, for a cache in 8 bits to its
        elements. Rows of no sequence, or whose position the tables do not hold
        (recorded), are not written to either; nor are keys and values that the
        pages have no room for (recorded)."""
        kind, dtype, index = self._type(q, "q"), q.dtype, self._index
        if q.dim() != 3 or q.shape[1] < 1:
            raise ValueError("q must be a %s [rows, heads, %d] tensor on %s" % (dtype, self.dim, self.device))
        heads = q.shape[1]
        qd = self._heads(q, "q", dtype, heads)
        kd, vd = self._heads(k, "k", dtype, self.kv_heads), self._heads(v, "v", dtype, self.kv_heads)
        self._layer(layer)
        rows = qd.n_rows
        if kd.n_rows != rows or vd.n_rows != rows:
            raise ValueError("q, k and v must have the same rows, k and v one shape, got %s, %s and %s"
                             % (tuple(q.shape), tuple(k.shape), tuple(v.shape)))
        table = cos.shape
        if len(table) != 2 or cos.dtype is not torch.float32 or cos.get_device() != index or not cos.is_contiguous() \
                or not 1 <= table[1] <= self.dim // 2 or table[0] < 1:
            raise ValueError("cos must be a contiguous fp32 [positions, up to %d] tensor on cuda:%d" % (self.dim // 2, index))
        if sin.shape != table or sin.dtype is not torch.float32 or sin.get_device() != index or not sin.is_contiguous():
            raise ValueError("sin must have cos' shape, type and device")
        forward_only(cos, "cos")
        forward_only(sin, "sin")
        at, n = self._seqs(seqs)
        if out is None:
            out = torch.empty_like(q, memory_format=torch.contiguous_format)
            od = _native.AimgHeads(out.data_ptr(), rows, heads * self.dim, self.dim, heads, self.dim)
        else:
            od = self._heads(out, "out", dtype, heads)
            if od.n_rows != rows:
                raise ValueError("out must have q's shape %s" % (tuple(q.shape),))
        launch(self._lib.aimg_cache_append_rotated, index, self._cache, self._scales_at, layer, qd, kd, vd, od, at,
               _int32(offsets, "offsets", (n + 1,), index), n,
               _native.AimgRotary(cos.data_ptr(), sin.data_ptr(), table[0], table[1], interleaved),
               None if positions is None else _int32(positions, "positions", (rows,), index), kind)
        return out

    def read(self, layer: int, seqs: torch.Tensor, offsets: torch.Tensor, rows: int, starts: torch.Tensor | None = None, *,
             dtype: torch.dtype | None = None, out: tuple[torch.Tensor, torch.Tensor] | None = None) -> tuple[torch.Tensor, torch.Tensor]:
        """Keys and values of a layer as packed rows [rows, kv_heads, dim], as
        prompt_attention takes them for a prompt that continues a context: rows
        offsets[b] .. offsets[b + 1] - 1 (int32, on the GPU; ``rows`` is their
        number) are positions starts[b] (int32, 0 where not given) and on of
        slot seqs[b]. They may pass its length, not its pages. dtype: bf16 or
        fp16 for a cache in 8 bits (bf16 where not given, and exact there), the
        pool's otherwise. Rows of no sequence, or of no page (recorded), are
        not written."""
        dtype = dtype or (self.pool.dtype if self.scales is None else torch.bfloat16)
        if dtype not in _TYPES or (self.scales is None and dtype is not self.pool.dtype):
            raise ValueError("dtype must be %s, got %s" % (self.pool.dtype if self.scales is None else "bf16 or fp16", dtype))
        self._layer(layer)
        if rows < 0:
            raise ValueError("rows must not be negative, got %d" % rows)
        if out is None:
            both = torch.empty((2, rows, self.kv_heads, self.dim), dtype=dtype, device=self.device)
            k, v = both.unbind(0)
            row = self.kv_heads * self.dim
            first = both.data_ptr()
            kd, vd = (_native.AimgHeads(at, rows, row, self.dim, self.kv_heads, self.dim) for at in (first, first + 2 * rows * row))
        else:
            k, v = out
            kd, vd = self._heads(k, "k", dtype, self.kv_heads), self._heads(v, "v", dtype, self.kv_heads)
            if kd.n_rows != rows or vd.n_rows != rows:
                raise ValueError("out must hold %d rows, got %d and %d" % (rows, kd.n_rows, vd.n_rows))
        at, n = self._seqs(seqs)
        launch(self._lib.aimg_cache_read, self._index, self._cache, self._scales_at, layer, at,
               _int32(offsets, "offsets", (n + 1,), self._index), None if starts is None else _int32(starts, "starts", (n,), self._index),
               n, kd, vd, _TYPES[dtype])
        return k, v

    def advance(self, seqs: torch.Tensor, offsets: torch.Tensor) -> None:
        """Slot seqs[b]'s length grows by offsets[b + 1] - offsets[b], the rows that were appended."""
        at, n = self._seqs(seqs)
        launch(self._lib.aimg_cache_advance, self._index, self._cache, at, _int32(offsets, "offsets", (n + 1,), self._index), n)

    def attend(self, layer: int, q: torch.Tensor, seqs: torch.Tensor, draft_offsets: torch.Tensor,
               masks: torch.Tensor | None = None, **options) -> torch.Tensor:
        """tree_attention of q over one layer of this cache; options are its keyword arguments (max_drafts is needed)."""
        if not -self.n_layers <= layer < self.n_layers:
            raise IndexError("layer %d is out of range for %d layers" % (layer, self.n_layers))
        pages, scales = self._described[layer]
        forward_only(self.pool, "pool")
        return attend(q, _query(q), pages, scales, self.pool.dtype, self._index, seqs, draft_offsets, masks, **options)

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
        entry = (self._lib.aimg_cache_commit, self._index, self._cache) if self.scales is None else \
            (self._lib.aimg_cache8_commit, self._index, self._cache, self._scales_at)
        launch(*entry, at, _int32(accepted, "accepted", (n, most), self._index), most,
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
        if self.scales is None:
            launch(self._lib.aimg_cache_fork, self._index, self._cache, s, d, n, work.data_ptr(), nbytes)
        else:
            launch(self._lib.aimg_cache8_fork, self._index, self._cache, self._scales_at, s, d, n, work.data_ptr(), nbytes)

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
        entry = (self._lib.aimg_cache_compact, self._index, self._cache) if self.scales is None else \
            (self._lib.aimg_cache8_compact, self._index, self._cache, self._scales_at)
        launch(*entry, _int32(table, "new_table", (self.max_seqs, self.max_pages), self._index),
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
