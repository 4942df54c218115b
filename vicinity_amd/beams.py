"""select_beams: the best continuations of a batch's beams by one token.

It stands beside KVCache: the rows that it returns are what ``KVCache.fork`` continues.
"""

from __future__ import annotations

import ctypes
import functools

import numpy as np

from . import _lib


@functools.lru_cache(maxsize=64)
def _workspace(*sizes) -> int:
    size = ctypes.c_size_t()
    _lib.check(_lib.load().vgpu_beams_workspace(*sizes, ctypes.byref(size)))
    return size.value


def select_beams(logits, scores, beams: int, k: int | None = None, stream=None):
    """The k best continuations of each group of `beams` rows by one token.

    logits [groups * beams, vocab], float32, float16 or bfloat16, any strides; scores float32
    [groups * beams], the rows' log-probabilities so far (None: 0).  A continuation's total is
    scores[row] + logits[row, token] - log(sum(exp(logits[row]))).  Returns (totals, rows,
    tokens), float32, int64 and int64 [groups, k], totals descending, of equal ones the lower
    row and then the lower token first (a row's larger logit, where float64 holds the totals as
    equal: a score of -1e30 leaves no difference); k None: beams.  With a cache that holds row i's tokens
    in sequence i, a step of beam search is ``cache.fork(rows.view(-1).tolist(), range(n))``
    with k = beams.

    Logits of -inf are tokens that cannot follow (a row of them, or a row whose score is -inf,
    has totals of -inf alone); a NaN or +inf among a row's logits or in its score makes all its
    totals NaN, which come first.  Totals are ordered in float64, from float32 exponentials, and
    rounded once.  At most 1024 beams and 256 results for a group.

    Queued on the current stream, or on `stream`, without waiting; it can be captured into a
    graph.  There is no backward."""
    import torch

    if not isinstance(logits, torch.Tensor) or logits.dtype not in (torch.float32, torch.float16, torch.bfloat16):
        raise TypeError("logits must be a float32, float16 or bfloat16 tensor")
    if logits.dim() != 2 or not logits.is_cuda:
        raise ValueError("logits must have the shape [rows, vocab], on a GPU")
    rows, vocab = logits.shape
    if scores is not None:
        if not isinstance(scores, torch.Tensor) or scores.dtype != torch.float32:
            raise TypeError("scores must be a float32 tensor")
        if scores.shape != (rows,) or scores.device != logits.device:
            raise ValueError(f"scores must have the shape [{rows}], on the logits' GPU")
    k = beams if k is None else k
    for name, value in (("beams", beams), ("k", k)):
        if not isinstance(value, (int, np.integer)) or not 0 < value < 1 << 31:
            raise ValueError(f"{name} must be an int above 0")
    beams, k = int(beams), int(k)
    dtype = 0 if logits.dtype == torch.float32 else 1 if logits.dtype == torch.float16 else 2
    size = _workspace(dtype, rows, vocab, beams, k)
    device = logits.device
    if stream is None and device.index == torch.cuda.current_device():
        return _select(torch, logits, scores, dtype, beams, k, size,
                       torch._C._cuda_getCurrentRawStream(device.index))
    use = torch.cuda.current_stream(device) if stream is None else stream
    with torch.cuda.device(device), torch.cuda.stream(use):
        for t in (logits, scores):
            if t is not None:
                t.record_stream(use)
        return _select(torch, logits, scores, dtype, beams, k, size, use.cuda_stream)


def _select(torch, logits, scores, dtype, beams, k, size, stream):
    device, (rows, vocab) = logits.device, logits.shape
    shape = (rows // beams, k)
    totals = torch.empty(shape, dtype=torch.float32, device=device)
    parents = torch.empty(shape, dtype=torch.int64, device=device)
    tokens = torch.empty(shape, dtype=torch.int64, device=device)
    work = torch.empty(size, dtype=torch.uint8, device=device)
    call = _lib.Beams(logits.data_ptr(), dtype, *logits.stride(), rows, vocab, beams, k,
                      None if scores is None else scores.data_ptr(),
                      0 if scores is None else scores.stride(0), work.data_ptr(), size,
                      totals.data_ptr(), parents.data_ptr(), tokens.data_ptr())
    _lib.check(_lib.load().vgpu_select_beams(ctypes.byref(call), stream or None))
    return totals, parents, tokens
