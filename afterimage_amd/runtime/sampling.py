"""Tokens from logits, on the GPU.

The reference's engine takes the largest logit of a pass
(afterimage/runtime/streaming_engine.py:2488-2600 verifies drafts against it);
a program that samples does so from what ``decompress_linear_gpu`` or
``decode_linear`` gives it. Work is ordered on the current stream and nothing
here synchronises or draws random numbers: they are arguments, so that a draw
can be repeated, and a verified tree's tokens follow the model's distribution
where a child is accepted if it is its parent's drawn token.
"""
from __future__ import annotations

import ctypes
import functools

import torch

from .. import _native
from .attention import forward_only, launch

MAX_VOCAB = 1 << 18
MAX_ROWS = 1 << 21

_TYPES = {torch.bfloat16: _native.AIMG_BF16, torch.float16: _native.AIMG_FP16, torch.float32: _native.AIMG_FP32}


def _vector(x: torch.Tensor, name: str, dtype: torch.dtype, rows: int, index: int) -> int:
    if x.dtype is not dtype or x.shape != (rows,) or x.get_device() != index or not x.is_contiguous():
        raise ValueError("%s must be a contiguous %s [%d] tensor on cuda:%d" % (name, dtype, rows, index))
    return x.data_ptr()


@functools.lru_cache(maxsize=1024)
def _workspace_nbytes(rows: int, vocab: int) -> int:
    nbytes = ctypes.c_size_t(0)
    _native.check(_native.lib().aimg_sample_workspace_nbytes(rows, vocab, ctypes.byref(nbytes)))
    return nbytes.value


def sample(logits: torch.Tensor, uniforms: torch.Tensor, *, temperature: float | torch.Tensor = 1.0,
           top_k: int | torch.Tensor = 0, top_p: float | torch.Tensor = 1.0, min_p: float | torch.Tensor = 0.0,
           logprobs: bool = False, out: torch.Tensor | None = None):
    """A token for each row of logits [rows, vocab] (bf16, fp16 or fp32, any
    row stride, vocab up to 2^18, up to 2^21 rows), from uniforms [rows] (fp32, in [0, 1)).

    A row's tokens stand in the order of falling logits, equal ones by rising
    index, and weigh w = exp((x - max) / temperature). Kept are those among the
    first top_k (0: all), in the shortest prefix whose weights reach top_p times
    the first top_k's (1: all), and with w >= min_p (0: all); the largest always.
    The token is the first whose weights, summed along the order, pass its
    uniform number times the sum of those kept. temperature 0 takes the
    largest's first token. Each setting is a number for all rows or a tensor
    [rows] on the GPU (fp32, top_k int32); a tensor's numbers out of range
    mean the nearest in it.

    Returns int64 tokens [rows] (out where given), with logprobs the
    logarithms (fp32) of the tokens' shares of the sums kept besides. Logits of
    -inf or NaN are no tokens; a row without any other gives -1 (and -inf).
    Results do not vary between calls. No gradients: logits or settings that
    require one are refused outside torch.no_grad()."""
    index, kind = logits.get_device(), _TYPES.get(logits.dtype)
    if index < 0:
        raise RuntimeError("sample runs on the GPU only; got logits on %s" % logits.device)
    if kind is None or logits.dim() != 2 or logits.shape[1] < 1 or (logits.stride(1) != 1 and logits.shape[1] > 1):
        raise ValueError("logits must be a bf16, fp16 or fp32 [rows, vocab] tensor, contiguous in its last dimension")
    rows, vocab = logits.shape
    if vocab > MAX_VOCAB:
        raise ValueError("logits: vocab must be at most %d, got %d" % (MAX_VOCAB, vocab))
    if rows > MAX_ROWS:
        raise ValueError("logits: at most %d rows, got %d" % (MAX_ROWS, rows))
    forward_only(logits, "logits")
    settings = _native.AimgSampling(temperature=1.0, top_p=1.0)
    for name, value, dtype, least, most in (("temperature", temperature, torch.float32, 0.0, None), ("top_k", top_k, torch.int32, 0, None),
                                            ("top_p", top_p, torch.float32, 0.0, 1.0), ("min_p", min_p, torch.float32, 0.0, 1.0)):
        if isinstance(value, torch.Tensor):
            forward_only(value, name)
            setattr(settings, name + "s", _vector(value, name, dtype, rows, index))
        elif not value >= least or (most is not None and value > most):
            raise ValueError("%s must be %s, got %r" % (name, "at least 0" if most is None else "in 0..1", value))
        else:
            setattr(settings, name, min(value, 0x7FFFFFFF) if name == "top_k" else float(value))
    uniforms_at = _vector(uniforms, "uniforms", torch.float32, rows, index)
    if out is None:
        out = torch.empty(rows, dtype=torch.int64, device=logits.device)
    out_at = _vector(out, "out", torch.int64, rows, index)
    logs = torch.empty(rows, dtype=torch.float32, device=logits.device) if logprobs else None
    nbytes = _workspace_nbytes(rows, vocab)
    # Held until the launches are made, from torch's allocator on the current stream.
    work = torch.empty(nbytes, dtype=torch.uint8, device=logits.device) if nbytes else None
    launch(_native.lib().aimg_sample, index, logits.data_ptr(), rows, logits.stride(0), vocab, kind, uniforms_at, settings, out_at,
           logs.data_ptr() if logprobs else None, work.data_ptr() if nbytes else None, nbytes)
    return (out, logs) if logprobs else out
