"""Two threads on streams of their own share a cache: pool, block table and workspaces."""

import threading

import pytest

from test_gpu_kv import _case, _rand, _torch

pytestmark = pytest.mark.gpu


def test_two_threads_get_what_one_gets():
    torch = _torch()
    _case("two threads, two streams, one cache")
    import vicinity_amd as va

    steps, heads, dim = 24, 2, 64
    k = [_rand((steps * 90, heads, dim), "bfloat16", 900 + t) for t in range(2)]
    v = [_rand((steps * 90, heads, dim), "bfloat16", 910 + t) for t in range(2)]
    q = [_rand((steps * 3, heads * 4, dim), "bfloat16", 920 + t) for t in range(2)]
    torch.cuda.synchronize()

    def go(cache, t, stream, out):
        with torch.cuda.stream(stream):
            for i in range(steps):
                cache.append(k[t][i * 90:(i + 1) * 90], v[t][i * 90:(i + 1) * 90], seqs=[t])
                got = cache.attend(q[t][i * 3:(i + 1) * 3], seqs=[t], counts=[3], decay=1.0)
                out.append((got, cache.read(seqs=[t])))
            stream.synchronize()

    def caches():
        return va.KVCache(2, heads, dim, 2 * steps * 3, block_tokens=32, max_blocks=steps * 3)

    alone = [[], []]
    one = caches()
    for t in range(2):
        go(one, t, torch.cuda.Stream(), alone[t])
    both, failed = [[], []], []
    shared = caches()

    def thread(t):
        try:
            go(shared, t, torch.cuda.Stream(), both[t])
        except Exception as e:  # noqa: BLE001 - reported below
            failed.append(e)

    threads = [threading.Thread(target=thread, args=(t,)) for t in range(2)]
    for x in threads:
        x.start()
    for x in threads:
        x.join(60)
    torch.cuda.synchronize()
    assert not failed, failed
    for t in range(2):
        assert len(both[t]) == steps
        for (a, held_a), (b, held_b) in zip(alone[t], both[t]):
            assert torch.equal(a, b)
            assert all(torch.equal(held_a[f], held_b[f]) for f in held_a)
