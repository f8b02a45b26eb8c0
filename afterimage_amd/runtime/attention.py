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
