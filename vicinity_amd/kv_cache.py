"""KVCache: a model's keys and values in HBM, in 8 bits with a scale for each block of
tokens and head, softmax attention over them, and eviction by accumulated weight.

It stands beside the indexes: what evict takes out of the cache are float32 keys and
values, and ``FlatIndex(dim, "cosine")`` ranks keys by the same inner product that the
attention takes them with.

Tensors are torch tensors on the cache's GPU.  Calls are queued on the current torch
stream, or on ``stream``, and return without waiting; a call on another stream than the
one before it waits for that one on the GPU.  Calls of several threads on one cache take
turns, on the host and on the GPU alike.  There is no backward: what enters the cache is
held without its gradient, and results have none.
"""

from __future__ import annotations

import contextlib
import ctypes
import math
import threading
from array import array

import numpy as np

from . import _lib

CODES = {"int8": 0, "fp8": 1}
FIELDS = ("k", "v", "positions", "weights")
_SAME = contextlib.nullcontext()  # the current stream


def _ptr(a: array) -> int:
    return a.buffer_info()[0]


def _array(kind: str, values, name: str) -> array:
    """Host integers for the library: a list, a range, an array ('i': 32 bits, 'q': 64)."""
    if not isinstance(values, (list, tuple, range)):
        values = np.asarray(values)
        if values.ndim != 1 or (values.size and values.dtype.kind not in "iu"):
            raise ValueError(f"{name} must be a 1-D array of integers")
        values = values.tolist()
    try:
        return array(kind, values)
    except (TypeError, OverflowError) as e:
        raise ValueError(f"{name} must be a 1-D array of integers that fit the library") from e


class KVCache:
    """num_seqs sequences over a pool of num_blocks blocks of block_tokens slots.

    code 'int8': value = code * scale, codes -127..127; 'fp8': e4m3 codes.  A sequence
    takes at most max_blocks blocks (None: all of them)."""

    def __init__(self, num_seqs: int, num_heads: int, head_dim: int, num_blocks: int,
                 block_tokens: int = 64, code: str = "int8", max_blocks: int | None = None):
        if code not in CODES:
            raise ValueError(f"code must be one of {sorted(CODES)}, got {code!r}")
        for name, value in (("num_seqs", num_seqs), ("num_heads", num_heads),
                            ("head_dim", head_dim), ("num_blocks", num_blocks),
                            ("block_tokens", block_tokens), ("max_blocks", max_blocks or 1)):
            if not 0 < int(value) < 1 << 31:
                raise ValueError(f"{name} must be in the range 1..2**31, got {value}")
        self._h = None
        self._L = _lib.load()
        params = _lib.KvParams(num_seqs, num_heads, head_dim, num_blocks, block_tokens,
                               max_blocks or 0, CODES[code])
        h = ctypes.c_void_p()
        _lib.check(self._L.vgpu_kv_new(ctypes.byref(params), ctypes.byref(h)))
        self._h = h
        self.num_seqs, self.num_heads, self.head_dim = num_seqs, num_heads, head_dim
        self.num_blocks, self.block_tokens, self.code = num_blocks, block_tokens, code
        import torch

        self.device = torch.device("cuda", torch.cuda.current_device())
        self._types = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
        self._all = array("i", range(num_seqs))
        # Held while a call reads the lengths, goes behind the last one's stream and queues its
        # work, so that two threads' calls reach the GPU in the order of their waits.
        self._turn = threading.Lock()
        self._last = None      # the stream of the last call, and its handle
        self._last_raw = None

    def __del__(self):
        h = getattr(self, "_h", None)
        if h is not None and h.value:
            self._L.vgpu_kv_free(h)
            self._h = None

    # ---- state ------------------------------------------------------------
    @property
    def lengths(self) -> np.ndarray:
        """Slots in use of every sequence, int64 [num_seqs]."""
        return np.array(self._lengths())

    def info(self) -> dict:
        """free_blocks, and device_bytes: the HBM that the cache holds."""
        out = _lib.KvInfo()
        _lib.check(self._L.vgpu_kv_get_info(self._h, ctypes.byref(out)))
        return {"free_blocks": out.free_blocks, "device_bytes": out.device_bytes}

    def truncate(self, lengths, seqs=None) -> None:
        """Forget each sequence's slots from lengths[i] on; 0 empties it.  A block that keeps
        slots keeps its scales, also one that a forgotten token raised, or made NaN."""
        ids = self._seqs(seqs)
        lens = self._ints(lengths, len(ids), "lengths")
        with self._turn:
            _lib.check(self._L.vgpu_kv_truncate(self._h, _ptr(ids), _ptr(lens), len(ids)))

    # ---- operators ----------------------------------------------------------
    def append(self, k, v, seqs=None, counts=None, positions=None, weights=None,
               stream=None) -> None:
        """Quantise new tokens behind those that the sequences hold.

        k, v [tokens, num_heads, head_dim], float32, float16 or bfloat16, any strides:
        counts[i] tokens of seqs[i] after those of seqs[i - 1] (seqs None: every
        sequence; counts None: the same number for each).  positions int32 and weights
        float32 [tokens, num_heads] are kept beside the slots (None: tokens counted from
        the sequence's start, and 0)."""
        ids = self._seqs(seqs)
        kt = self._tensor(k, "k", self.num_heads)
        vt = self._tensor(v, "v", self.num_heads)
        if k.shape != v.shape or k.dtype != v.dtype:
            raise ValueError("k and v must have the same shape and dtype")
        n = self._counts(counts, len(ids), k.shape[0])
        pos = self._side(positions, "positions", k.shape[0], "int32")
        wts = self._side(weights, "weights", k.shape[0], "float32")
        with self._turn:
            s, _ = self._stream(stream, (k, v, positions, weights))
            _lib.check(self._L.vgpu_kv_append(self._h, _ptr(ids), _ptr(n), len(ids),
                                              ctypes.byref(kt), ctypes.byref(vt), pos, wts, s))

    def attend(self, q, seqs=None, counts=None, scale: float | None = None, causal: bool = True,
               window: int = 0, mask=None, decay: float | None = None, out=None,
               return_lse: bool = False, stream=None):
        """softmax(scale * q k^T) v over the cached slots, [tokens, heads, head_dim].

        q [tokens, heads, head_dim] belongs to the last counts[i] tokens of seqs[i];
        heads is a multiple of num_heads, consecutive query heads share a key/value head.
        Token i stands at slot len - counts + i and sees the slots up to its own (causal;
        else all), of them the last `window` (0: all), of them those where mask
        [tokens, slots] (bool) is set.  A token that sees nothing gets 0 and lse -inf.
        scale None: 1 / sqrt(head_dim).  decay: the accumulated weight of a slot and head
        becomes decay * weight + what the call's tokens gave it (None: weights stay).
        return_lse: also the float32 logarithms of the softmax denominators
        [tokens, heads].

        Sums, logarithms and weights are float32.  16-bit queries are taken exactly and
        their probabilities multiply the values with 11 bits; float32 queries with 22 bits
        of their row's largest element, and so the probabilities; what is below 2^-30 of
        the largest adds nothing to the result.  Scores (scale * q k) are float32: they have
        to stay below 2^24."""
        import torch

        ids = self._seqs(seqs)
        qt = self._tensor(q, "q", None)
        tokens, heads = q.shape[0], q.shape[1]
        if heads == 0 or heads % self.num_heads:
            raise ValueError(f"q has {heads} heads, not a multiple of the cache's "
                             f"{self.num_heads}")
        n = self._counts(counts, len(ids), tokens)
        if not isinstance(window, (int, np.integer)) or window < 0:
            raise ValueError("window must be an int, 0 or more")
        if out is not None and (out.shape != q.shape or out.dtype != q.dtype
                                or out.device != q.device or not out.is_contiguous()):
            raise ValueError("out must be contiguous, of q's shape, dtype and device")
        if mask is not None:
            if mask.dtype not in (torch.bool, torch.uint8) or mask.dim() != 2 \
                    or mask.shape[0] != tokens or mask.device != self.device:
                raise ValueError("mask must be a bool or uint8 tensor [tokens, slots] on the "
                                 "cache's GPU")
        with self._turn:
            s, ctx = self._stream(stream, (q, mask, out))
            with ctx:
                if out is None:
                    out = torch.empty_like(q, memory_format=torch.contiguous_format)
                lse = q.new_empty((tokens, heads), dtype=torch.float32) if return_lse else None
            query = _lib.KvQuery(
                qt, heads, 1.0 / math.sqrt(self.head_dim) if scale is None else scale, int(causal),
                min(int(window), 1 << 62), mask.data_ptr() if mask is not None else None,
                mask.stride(0) if mask is not None else 0, mask.stride(1) if mask is not None else 0,
                mask.shape[1] if mask is not None else 0, int(decay is not None),
                0.0 if decay is None else decay, out.data_ptr(),
                lse.data_ptr() if lse is not None else None)
            _lib.check(self._L.vgpu_kv_attend(self._h, _ptr(ids), _ptr(n), len(ids),
                                              ctypes.byref(query), s))
        return (out, lse) if return_lse else out

    def evict(self, budget: int, recent: int = 0, seqs=None, into=None, dropped: bool = False,
              stream=None):
        """Cut each sequence longer than `budget` slots down to it.

        Every head keeps its last `recent` slots and those of largest accumulated weight
        among the others (of equal ones the lower slot), in their order.  into: empty
        sequences that receive the result (seqs stay as they are); None: in place.
        dropped: return what leaves as a dict, positions int32 [n, most, num_heads]
        (-1 where a sequence lost fewer), k and v float32 [n, most, num_heads, head_dim]
        (zeros there)."""
        import torch

        ids = self._seqs(seqs)
        to = None if into is None else self._seqs(into)
        if to is not None and len(to) != len(ids):
            raise ValueError(f"into names {len(to)} sequences, seqs {len(ids)}")
        for name, value in (("budget", budget), ("recent", recent)):
            if not isinstance(value, (int, np.integer)) or not 0 <= value < 1 << 30:
                raise ValueError(f"{name} must be an int from 0 to 2**30 - 1")
        with self._turn:
            s, ctx = self._stream(stream, ())
            gone, most = None, 0
            if dropped:
                lens = self._lengths()
                most = max(max((lens[i] for i in ids), default=0) - int(budget), 0)
                shape = (len(ids), most, self.num_heads)
                with ctx:
                    gone = {"positions": torch.empty(shape, dtype=torch.int32, device=self.device),
                            "k": torch.empty(shape + (self.head_dim,), device=self.device,
                                             dtype=torch.float32)}
                    gone["v"] = torch.empty_like(gone["k"])
            ptr = [gone[f].data_ptr() if gone and most else None for f in ("positions", "k", "v")]
            _lib.check(self._L.vgpu_kv_evict(self._h, _ptr(ids),
                                             None if to is None else _ptr(to), len(ids), budget,
                                             recent, most, *ptr, s))
        return gone

    def fork(self, seqs, into, lengths=None, copy: bool = False, stream=None) -> None:
        """Each sequence into[i] becomes a continuation of its own of the first lengths[i] slots
        of seqs[i] (None: all) as they stood before the call; what it held is forgotten.

        into are different sequences; one of seqs may be continued by several, and be among
        into: a step of beam search is ``fork(parents, beams)``.  Blocks are shared, and copied
        when a holder writes into one that others hold too (append into a begun block, attend
        with decay); copy=True: copied at once.  Both need free blocks for the copies.  Either
        way each sequence reads, attends and changes as if it were alone; attend
        without decay reads what several sequences share once for all, where that is faster."""
        to, part = self._seqs(into), self._slice(seqs)
        # (the library checks their range)
        ids = _array("i", seqs, "sequences") if part is None else self._all[part]
        if len(ids) != len(to):
            raise ValueError(f"into names {len(to)} sequences, seqs {len(ids)}")
        lens = None if lengths is None else self._ints(lengths, len(ids), "lengths")
        with self._turn:
            s, _ = self._stream(stream, ())
            _lib.check(self._L.vgpu_kv_fork(self._h, _ptr(ids), _ptr(to),
                                            None if lens is None else _ptr(lens), len(ids),
                                            int(bool(copy)), s))

    def compact(self, num_blocks: int | None = None, stream=None) -> int:
        """Move the used blocks to the front of the pool; returns how many moved.  num_blocks:
        to a pool of so many blocks, not fewer than are used, in place of the old one, whose
        memory is given back (both exist during the call, which then waits for the GPU)."""
        if num_blocks is not None and not (isinstance(num_blocks, (int, np.integer))
                                           and 0 < num_blocks <= 1 << 30):
            raise ValueError("num_blocks must be an int from 1 to 2**30")
        moved = ctypes.c_size_t()
        with self._turn:
            s, _ = self._stream(stream, ())
            _lib.check(self._L.vgpu_kv_compact(self._h, num_blocks or 0, ctypes.byref(moved), s))
            self.num_blocks = int(num_blocks or self.num_blocks)
        return moved.value

    def read(self, seqs=None, first=None, counts=None, fields=FIELDS, dtype=None,
             stream=None) -> dict:
        """What the slots first[i] .. first[i] + counts[i] - 1 of seqs[i] hold (None: from
        0, to the end), one sequence after the other: 'k' and 'v' [tokens, num_heads,
        head_dim] in dtype (None: float32), 'positions' int32 and 'weights' float32
        [tokens, num_heads]."""
        import torch

        dtype = torch.float32 if dtype is None else dtype
        if dtype not in self._types:
            raise TypeError("dtype must be float32, float16 or bfloat16")
        for f in fields:
            if f not in FIELDS:
                raise ValueError(f"fields must be among {FIELDS}")
        ids = self._seqs(seqs)
        at = self._ints(0 if first is None else first, len(ids), "first")
        if first is not None and at and min(at) < 0:
            raise ValueError("first must not be negative")
        with self._turn:
            if counts is None:  # to the end; the library checks what the tensors were sized by
                lens = self._lengths()
                part = self._slice(seqs)
                n = lens if ids is self._all else lens[part] if part is not None else \
                    array("q", map(lens.__getitem__, ids))
                if first is not None and n:
                    left = np.frombuffer(n, np.int64)  # n's own memory
                    np.subtract(left, at, out=left)
            else:
                n = self._ints(counts, len(ids), "counts")
            tokens = max(sum(n), 0)
            s, ctx = self._stream(stream, ())
            types = {"positions": torch.int32, "weights": torch.float32}
            res = {}
            with ctx:
                for f in fields:
                    shape = (tokens, self.num_heads) + ((self.head_dim,) if f in "kv" else ())
                    res[f] = torch.empty_like(res["k"]) if f == "v" and "k" in res else \
                        torch.empty(shape, dtype=types.get(f, dtype), device=self.device)
            ptr = [res[f].data_ptr() if f in res else None for f in FIELDS]
            _lib.check(self._L.vgpu_kv_read(self._h, _ptr(ids), _ptr(at), _ptr(n), len(ids),
                                            self._types[dtype], *ptr, s))
        return res

    # ---- arguments ------------------------------------------------------------
    def _lengths(self) -> array:
        out = array("q", bytes(8 * self.num_seqs))
        _lib.check(self._L.vgpu_kv_lengths(self._h, _ptr(out)))
        return out

    def _slice(self, seqs) -> slice | None:
        """An ascending range of the cache's sequences as a slice of all; anything else None."""
        if type(seqs) is range and seqs.step > 0 and 0 <= seqs.start <= seqs.stop <= self.num_seqs:
            return slice(seqs.start, seqs.stop, seqs.step)
        return None

    def _seqs(self, seqs) -> array:
        if seqs is None:
            return self._all
        part = self._slice(seqs)
        if part is not None:
            return self._all[part]
        a = _array("i", seqs, "sequences")
        if a and not 0 <= min(a) <= max(a) < self.num_seqs:
            raise ValueError(f"sequence out of range [0, {self.num_seqs})")
        return a

    @staticmethod
    def _ints(values, n: int, name: str) -> array:
        if isinstance(values, (int, np.integer)):
            return _array("q", (int(values),), name) * n
        a = _array("q", values, name)
        if len(a) != n:
            raise ValueError(f"{name} must have one entry for each of the {n} sequences")
        return a

    def _counts(self, counts, n: int, tokens: int) -> array:
        if counts is None:
            if n == 0 or tokens % n:
                raise ValueError(f"{tokens} tokens cannot be shared out to {n} sequences: "
                                 "counts is needed")
            return array("q", [tokens // n]) * n
        a = self._ints(counts, n, "counts")
        if (a and min(a) < 0) or sum(a) != tokens:
            raise ValueError(f"counts must add up to the {tokens} tokens given")
        return a

    def _tensor(self, t, name: str, heads):
        import torch

        if not isinstance(t, torch.Tensor):
            raise TypeError(f"{name} must be a torch tensor")
        if t.dtype not in self._types:
            raise TypeError(f"{name} must be float32, float16 or bfloat16")
        if t.dim() != 3 or t.shape[2] != self.head_dim or (heads and t.shape[1] != heads):
            raise ValueError(f"{name} must have the shape [tokens, {heads or 'heads'}, "
                             f"{self.head_dim}], got {list(t.shape)}")
        if t.device != self.device:
            raise ValueError(f"{name} must be on the cache's GPU ({self.device})")
        return _lib.KvTensor(t.data_ptr() or None, self._types[t.dtype], *t.stride())

    def _side(self, t, name: str, tokens: int, dtype: str):
        import torch

        if t is None:
            return None
        if not isinstance(t, torch.Tensor) or t.dtype != getattr(torch, dtype):
            raise TypeError(f"{name} must be a torch tensor of {dtype}")
        if t.shape != (tokens, self.num_heads) or t.device != self.device \
                or not t.is_contiguous():
            raise ValueError(f"{name} must be contiguous, [tokens, {self.num_heads}], on the "
                             "cache's GPU")
        return t.data_ptr()

    def _stream(self, stream, tensors):
        """The call's stream handle and a context that allocates on it.  Puts the call
        behind the last one and keeps the tensors' memory until it has run."""
        import torch

        if stream is None:
            raw = torch._C._cuda_getCurrentRawStream(self.device.index)
            if raw == self._last_raw:
                return raw or None, _SAME
            use = torch.cuda.current_stream(self.device)
        else:
            use, raw = stream, stream.cuda_stream
        with torch.cuda.stream(use):
            capturing = torch.cuda.is_current_stream_capturing()  # refused by the library
        if not capturing:
            if self._last is not None and self._last_raw != raw:
                use.wait_stream(self._last)
            self._last, self._last_raw = use, raw
        if stream is None or torch.cuda.current_stream(self.device) == use:
            return raw or None, _SAME
        for t in tensors:
            if t is not None:
                t.record_stream(use)
        return raw or None, torch.cuda.stream(use)
