"""KVCache against a library that keeps lengths and notes what it is asked to do, no GPU: calls
of several threads on one handle, and integers that the C interface cannot hold."""

import ctypes
import threading
import types

import numpy as np
import pytest

torch = pytest.importorskip("torch")


class Library:
    """Lengths, and the calls in the order in which they arrive."""

    def __init__(self, lengths):
        self.lengths = list(lengths)
        self.calls = []
        self.streams = []  # ("call", stream) and ("wait", stream, for that one)
        self.after_lengths = None  # what another thread does next

    def vgpu_kv_new(self, params, out):
        return 0

    def vgpu_kv_lengths(self, h, out):
        for i, n in enumerate(self.lengths):
            ctypes.c_int64.from_address(out + 8 * i).value = n
        if self.after_lengths:
            self.after_lengths()
        return 0

    def vgpu_kv_read(self, h, ids, first, counts, n, dtype, k, v, pos, wts, stream):
        ids = np.ctypeslib.as_array(ctypes.cast(ids, ctypes.POINTER(ctypes.c_int32)), (n,))
        first = np.ctypeslib.as_array(ctypes.cast(first, ctypes.POINTER(ctypes.c_int64)), (n,))
        if counts is None:  # to the end, as the library counts it
            rows = sum(self.lengths[i] - f for i, f in zip(ids, first))
        else:
            rows = np.ctypeslib.as_array(ctypes.cast(counts, ctypes.POINTER(ctypes.c_int64)), (n,)).sum()
        self.calls.append(("read", int(rows)))
        self.streams.append(("call", stream or 0))
        return 0

    def vgpu_kv_evict(self, h, ids, into, n, budget, recent, dropped, dpos, dk, dv, stream):
        self.calls.append(("evict", ctypes.c_size_t(budget).value, ctypes.c_size_t(recent).value))
        return 0

    def vgpu_kv_attend(self, h, ids, counts, n, query, stream):
        self.calls.append(("attend", query._obj.window))
        return 0


@pytest.fixture
def cache(monkeypatch):
    import vicinity_amd as va
    from vicinity_amd import _lib

    lib = Library([5, 0, 7])
    monkeypatch.setattr(_lib, "load", lambda: lib)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda index: 0, raising=False)
    monkeypatch.setattr(torch.cuda, "current_stream",
                        lambda device=None: types.SimpleNamespace(cuda_stream=0, wait_stream=lambda other: None))
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)

    class On:
        def __init__(self, stream):
            pass

        def __enter__(self):
            return self

        def __exit__(self, *exc):
            return False

    monkeypatch.setattr(torch.cuda, "stream", On)
    c = va.KVCache(3, 2, 4, 16)
    c.device = torch.device("cpu")
    return c, lib


@pytest.mark.parametrize("seqs,first", [(None, None), ([2, 0], [3, 1]), ([0], 2)])
@pytest.mark.parametrize("change", [+3, -2])
def test_read_to_the_end_writes_as_many_rows_as_it_allocated(cache, seqs, first, change):
    """Another thread appends to, or truncates, sequence 0 once the tensors' size is known."""
    c, lib = cache

    def other():
        lib.after_lengths = None
        lib.lengths[0] += change

    lib.after_lengths = other
    got = c.read(seqs=seqs, first=first)
    assert lib.calls == [("read", got["k"].shape[0])]


class Stream:
    def __init__(self, lib, number, hold=None):
        self.lib, self.cuda_stream, self.hold = lib, number, hold

    def wait_stream(self, other):
        if self.hold:
            self.hold()
        self.lib.streams.append(("wait", self.cuda_stream, other.cuda_stream))


def test_calls_of_two_threads_on_two_streams_follow_one_another(cache):
    """While the first thread's stream is put behind the last call, a second thread calls: what
    each thread queues must lie behind what the library was given before it."""
    c, lib = cache
    c.read()
    second = threading.Thread(target=lambda: c.read(stream=Stream(lib, 2)))

    def hold():
        second.start()
        second.join(0.5)  # time enough to get past the first thread, if nothing keeps it

    c.read(stream=Stream(lib, 1, hold))
    second.join()
    calls = [i for i, e in enumerate(lib.streams) if e[0] == "call"]
    assert sorted(lib.streams[i][1] for i in calls) == [0, 1, 2]
    for a, b in zip(calls, calls[1:]):
        assert ("wait", lib.streams[b][1], lib.streams[a][1]) in lib.streams[a:b], lib.streams


def test_read_refuses_a_negative_first_before_it_allocates(cache):
    c, lib = cache
    with pytest.raises(ValueError, match="first"):
        c.read(first=[0, 0, -(1 << 62)])
    assert not lib.calls


@pytest.mark.parametrize("name", ["budget", "recent"])
@pytest.mark.parametrize("value", [1 << 30, (1 << 64) + 5, (1 << 64) - 1])
def test_budgets_beyond_the_interface_are_refused(cache, name, value):
    """2^64 + 5 would arrive as 5, and cut every sequence to 5 slots."""
    c, lib = cache
    with pytest.raises(ValueError, match=name):
        c.evict(**({"budget": 8, "recent": 0} | {name: value}))
    assert not lib.calls
    c.evict((1 << 30) - 1, np.int64(4))
    assert lib.calls == [("evict", (1 << 30) - 1, 4)]


@pytest.mark.parametrize("window,arrives", [(0, 0), (7, 7), (np.int32(9), 9), (1 << 31, 1 << 31),
                                            ((1 << 64) + 1, 1 << 62), (1 << 64, 1 << 62)])
def test_a_window_beyond_the_interface_is_as_good_as_none(cache, window, arrives):
    c, lib = cache
    c.attend(torch.zeros((3, 2, 4)), counts=[1, 1, 1], window=window)
    assert lib.calls == [("attend", arrives)]
