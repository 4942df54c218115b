"""Numbers at the C entry that no call can have: refused on the host, before anything is queued."""

import ctypes

import numpy as np
import pytest

from test_gpu_kv import _case, _rand, _torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("counts", [[1 << 62], [(1 << 62) + 1], [1 << 61, 1 << 61, 1], [(1 << 63) - 1], [-1],
                                    [1 << 28], [1, -(1 << 63)]])
def test_token_counts_whose_rows_wrap_around(counts):
    """2^62 tokens of 4 heads are 2^64 rows, 0 as a 64-bit number."""
    torch = _torch()
    _case(f"counts {counts}")
    import vicinity_amd as va
    from vicinity_amd import _lib

    n = len(counts)
    cache = va.KVCache(n, 4, 64, 2 * n, block_tokens=32)
    x = _rand((4 * n, 4, 64), "bfloat16", 500)
    cache.append(x, x)
    q = _rand((n, 4, 64), "bfloat16", 501)
    want = cache.attend(q)
    out = torch.zeros_like(q)
    ids, c = np.arange(n, dtype=np.int32), np.array(counts, np.int64)
    query = _lib.KvQuery(_lib.KvTensor(q.data_ptr(), 2, *q.stride()), 4, 0.125, 1, 0, None, 0, 0, 0, 0, 0.0,
                         out.data_ptr(), None)
    with pytest.raises(ValueError, match="counts|rows"):
        _lib.check(cache._L.vgpu_kv_attend(cache._h, ids.ctypes.data_as(ctypes.c_void_p),
                                           c.ctypes.data_as(ctypes.c_void_p), n, ctypes.byref(query), None))
    torch.cuda.synchronize()
    assert not out.any() and torch.equal(cache.attend(q), want)
