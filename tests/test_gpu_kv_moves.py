"""Block copies: positions and weights of every slot and head, whatever the pieces that a block's
codes are cut into and the shares of the slots that go with each."""

import pytest

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("heads,block,dim", [
    (1, 32, 40), (3, 32, 250), (5, 128, 80), (7, 64, 192), (11, 256, 128), (64, 256, 64), (33, 256, 256)])
def test_positions_and_weights_of_all_slots(heads, block, dim):
    import torch

    import vicinity_amd as va

    print(f"[case] kv moves: {heads} heads, blocks of {block}, dim {dim}", flush=True)
    n, lens = 3, [2 * block + 5, 1, 3 * block]
    t, blocks = sum(lens), 3 + 1 + 3
    g = torch.Generator().manual_seed(heads)
    k, v = (torch.randn((t, heads, dim), generator=g).to("cuda:0") for _ in range(2))
    w = torch.rand((t, heads), generator=g).to("cuda:0")
    p = torch.randint(0, 1 << 30, (t, heads), generator=g, dtype=torch.int32).to("cuda:0")
    cache = va.KVCache(2 * n, heads, dim, 2 * blocks, block_tokens=block)
    cache.append(k, v, seqs=range(n), counts=lens, positions=p, weights=w)
    want = cache.read(seqs=range(n))
    assert torch.equal(want["positions"], p) and torch.equal(want["weights"], w)

    def same(seqs):
        got = cache.read(seqs=seqs)
        for f in want:
            assert torch.equal(got[f], want[f]), f

    cache.fork(range(n), range(n, 2 * n), copy=True)
    same(range(n, 2 * n))
    cache.truncate([0] * n, seqs=range(n))
    assert cache.compact() == blocks
    same(range(n, 2 * n))
    assert cache.compact(blocks + 2) == blocks
    same(range(n, 2 * n))
