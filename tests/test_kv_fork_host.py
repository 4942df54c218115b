"""Forks and compaction without a GPU: refusals that come before any device call."""

import ctypes

import pytest


def test_null_handles_are_refused():
    from vicinity_amd import _lib

    lib, ids = _lib.load(), (ctypes.c_int32 * 1)()
    at = ctypes.addressof(ids)
    for call in (lambda: lib.vgpu_kv_fork(None, at, at, None, 1, 0, None),
                 lambda: lib.vgpu_kv_fork(None, None, None, None, 0, 1, None),
                 lambda: lib.vgpu_kv_compact(None, 0, None, None),
                 lambda: lib.vgpu_test_set_kv_shared_bytes(None, 0)):
        assert call() == _lib.ERR_INVALID_PARAMETER
        assert b"null" in lib.vgpu_last_error()


@pytest.mark.parametrize("seqs", [range(0), range(5), range(2, 5), range(1, 5, 3), range(4, -1, -1), range(4, 0, -2),
                                  range(0, -1), range(3, 1), range(7, 7), range(1, 7, 4)])
def test_ranges_name_the_sequences_that_lists_name(seqs):
    from array import array

    from vicinity_amd import KVCache

    cache = KVCache.__new__(KVCache)
    cache.num_seqs, cache._all, cache._h = 6, array("i", range(6)), None
    assert list(cache._seqs(seqs)) == list(seqs) == list(cache._seqs(list(seqs)))
    assert len(cache._all) == 6


@pytest.mark.parametrize("seqs", [range(7), range(6, 7), range(-1, 3), range(6, 0, -1), range(2, 8, 5), range(-3, -1)])
def test_ranges_outside_the_cache_are_refused(seqs):
    from array import array

    from vicinity_amd import KVCache

    cache = KVCache.__new__(KVCache)
    cache.num_seqs, cache._all, cache._h = 6, array("i", range(6)), None
    with pytest.raises(ValueError, match="out of range"):
        cache._seqs(seqs)
