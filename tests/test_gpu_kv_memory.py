"""Workspaces of the attention memory that grow while the device has little memory left."""

import pytest

from test_gpu_kv import _case, _rand, _torch

pytestmark = pytest.mark.gpu


def test_a_workspace_grows_by_what_it_needs_where_there_is_no_more():
    """The first allocation of a call fails; what the call needs still fits."""
    torch = _torch()
    _case("a larger step of a workspace does not fit")
    import vicinity_amd as va
    from vicinity_amd import _lib

    n, more = 20_011, 1000
    x = _rand((n + more, 2, 64), "bfloat16", 400)
    q = _rand((1, 4, 64), "bfloat16", 401)
    cache = va.KVCache(1, 2, 64, 400)
    cache.append(x[:n], x[:n])
    cache.attend(q)
    cache.append(x[n:], x[n:])
    lib = _lib.load()
    for fails, works in ((1, True), (1, True), (50, False)):
        # (the third call needs a workspace that is not there yet: scores)
        _lib.check(lib.vgpu_test_fail_device_allocations(0, fails))
        try:
            if works:
                out = cache.attend(q)
            else:
                with pytest.raises(_lib.VicinityGpuError) as e:
                    cache.attend(q, decay=1.0)
                assert e.value.code == _lib.ERR_OUT_OF_MEMORY
        finally:
            _lib.check(lib.vgpu_test_fail_device_allocations(0, 0))
    fresh = va.KVCache(1, 2, 64, 400)
    fresh.append(x[:n], x[:n])
    fresh.append(x[n:], x[n:])
    assert torch.equal(out, fresh.attend(q))
    assert torch.equal(cache.attend(q, decay=1.0), out)
