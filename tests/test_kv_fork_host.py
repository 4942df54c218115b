"""Forks and compaction without a GPU: refusals that come before any device call."""

import ctypes


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
