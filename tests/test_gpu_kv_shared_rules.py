"""Which way attention of forks goes: by 16 rows, by many rows, or each sequence by itself; around
the sizes where that changes, against the definition in 64 bits."""

import numpy as np
import pytest

from test_gpu_kv import _rand
from test_gpu_kv_shared import _check_large, _large, share

pytestmark = pytest.mark.gpu


def _case(msg):
    print(f"[case] kv shared rules: {msg}", flush=True)


# forks, query heads to a head, slots: (forks * group / 16) * 8 heads * slots / 32 tiles of 16 rows
@pytest.mark.parametrize("dim,dtype", [(64, "bfloat16"), (64, "float32"), (96, "float16"), (128, "bfloat16"),
                                       (128, "float32"), (192, "bfloat16"), (192, "float32"), (256, "float16")])
@pytest.mark.parametrize("forks,group,slots", [(61, 4, 16_352), (61, 4, 16_384), (37, 7, 33_000)])
def test_around_the_tiles_of_the_kernel_of_many_rows(dim, dtype, forks, group, slots):
    _case(f"{dim} {dtype} {forks} x {group} rows over {slots}")
    cache = _large(slots, [5 + i % 3 for i in range(forks)], 8, dim, 64, "int8", dtype)
    q = _rand((forks, 8 * group, dim), dtype, 7)
    _check_large(cache, q, list(range(1, forks + 1)), [1] * forks)


def usual(cache):
    """Shared slots are read once where a program's calls do so."""
    from vicinity_amd import _lib

    _lib.check(_lib.load().vgpu_test_set_kv_shared_bytes(cache._h, 8 << 20))
    return cache


# Calls that take each sequence by itself, so forks come out bit for bit as copies do: sequences
# whose rows fill tiles by themselves, and those that the kernel of many rows takes alone.
@pytest.mark.parametrize("forks,tokens,group,prefix,heads,dim,dtype", [
    (32, 5, 4, 2048, 8, 128, "bfloat16"),    # 20 rows each, 512 workgroups of 16 rows
    (32, 20, 4, 2048, 8, 64, "float16"),     # 80 rows
    (61, 4, 4, 4096, 8, 256, "bfloat16"),    # 16 rows, a dimension that has no kernel for many
    (64, 1, 4, 960, 8, 128, "bfloat16"),     # 512 workgroups that need no split, few slots shared
    (128, 1, 1, 1900, 4, 64, "float32"),     # the same in two launches
    (5, 1, 8, 1312, 8, 128, "bfloat16"),     # 10.7 MB that would be left unread
    (8, 64, 4, 4096, 8, 128, "bfloat16"),    # 256 rows: two workgroups of many rows, full
    (2, 512, 4, 8192, 8, 128, "float32"),
    (2, 2048, 4, 2048, 8, 192, "bfloat16")])
def test_forks_with_rows_of_their_own_are_taken_as_copies_are(forks, tokens, group, prefix, heads, dim, dtype):
    import torch

    import vicinity_amd as va

    _case(f"{forks} forks x {tokens} tokens x {group}, {prefix} slots of {heads} x {dim}, {dtype}")
    blocks = forks * (-(-(prefix + tokens) // 64) + 1) + prefix // 64
    cache = va.KVCache(forks + 1, heads, dim, blocks, code="int8")
    k, v = (_rand((prefix, heads, dim), dtype, i) for i in (1, 2))
    nk, nv = (_rand((forks * tokens, heads, dim), dtype, i) for i in (3, 4))
    q = _rand((forks * tokens, heads * group, dim), dtype, 5)
    got = []
    for copy in (False, True):
        cache.truncate(0)
        cache.append(k, v, seqs=[forks])
        cache.fork([forks] * forks, range(forks), copy=copy)
        cache.append(nk, nv, seqs=range(forks))
        got.append(cache.attend(q, seqs=range(forks), return_lse=True))
    for a, b in zip(*got):
        assert torch.equal(a, b)


@pytest.mark.parametrize("dim,dtype", [(64, "bfloat16"), (80, "float32"), (128, "float16"), (256, "bfloat16")])
def test_many_tokens_and_single_ones_of_the_same_prefix(dim, dtype):
    """A prompt that comes in beside answers that go on: only the answers share tiles."""
    cache = usual(_large(4100, [700, 3, 40, 9, 1, 64, 65, 300], 8, dim, 64, "fp8", dtype))
    counts = [700, 1, 1, 5, 1, 1, 30, 257]
    _case(f"{dim} {dtype}")
    q = _rand((sum(counts), 8 * 4, dim), dtype, 7)
    for window in (0, 3000):
        _check_large(cache, q, list(range(1, 9)), counts, window=window)
    # all of them alike, and none of them
    share(cache)
    _check_large(cache, q, list(range(1, 9)), counts)
    _check_large(usual(cache), q[:8], list(range(1, 9)), [1] * 8)


def test_groups_of_which_one_or_none_is_left():
    """Of each prompt's answers all but one, or all, are taken by themselves."""
    import torch

    import vicinity_amd as va

    cache = va.KVCache(12, 8, 128, 2000, code="int8")
    k, v = (_rand((8192, 8, 128), "bfloat16", i) for i in (1, 2))
    cache.append(k, v, seqs=[10, 11], counts=[4096, 4096])
    cache.fork([10] * 5 + [11] * 5, range(10))
    counts = [1, 150, 200, 170, 260, 99, 180, 140, 300, 210]
    k, v = (_rand((sum(counts), 8, 128), "bfloat16", i) for i in (3, 4))
    cache.append(k, v, seqs=range(10), counts=counts)
    q = _rand((sum(counts), 32, 128), "bfloat16", 5)
    _check_large(cache, q, list(range(10)), counts)
    alone = torch.cat([cache.attend(q[sum(counts[:i]):sum(counts[:i + 1])], seqs=[i]) for i in range(10)])
    whole = cache.attend(q, seqs=range(10), counts=counts)
    assert (alone - whole).abs().max() <= 2.0 ** -6 * whole.abs().max()


@pytest.mark.parametrize("dim,dtype,window", [(64, "bfloat16", 0), (128, "float32", 0), (96, "float16", 700), (256, "bfloat16", 0)])
def test_sequences_that_share_nothing_beside_those_that_do(dim, dtype, window):
    """Sequences in no group, an empty one and one without tokens among them, in a call of forks."""
    import torch

    import vicinity_amd as va

    _case(f"{dim} {dtype} window {window}")
    heads, group = 8, 4
    cache = va.KVCache(24, heads, dim, 800, code="int8")
    k, v = (_rand((9000, heads, dim), dtype, i) for i in (1, 2))
    cache.append(k, v, seqs=[20, 21], counts=[8800, 200])
    cache.fork([20] * 9 + [21] * 3, range(12))
    own = [5, 1, 64, 7, 33, 2, 90, 1, 12, 3, 4, 5]
    alone = [1, 100, 300, 32]
    k, v = (_rand((sum(own + alone), heads, dim), dtype, i) for i in (3, 4))
    cache.append(k, v, seqs=list(range(12)) + [12, 13, 14, 15], counts=own + alone)
    seqs, counts = [12, 3, 16, 0, 1, 9, 17, 2, 4, 10, 5, 13, 6, 7, 8, 11, 14, 15], [1] * 18
    counts[4], counts[6] = 4, 0  # (17: empty, and without tokens; 16: empty)
    q = _rand((sum(counts), heads * group, dim), dtype, 5)
    for shared in (share, usual):
        shared(cache)
        out, lse = cache.attend(q, seqs=seqs, counts=counts, window=window, return_lse=True)
        assert (out[2] == 0).all() and torch.isneginf(lse[2]).all()
        live = [i for i, s in enumerate(seqs) if s not in (16, 17)]
        rows = torch.cat([torch.arange(sum(counts[:i]), sum(counts[:i + 1])) for i in live]).to("cuda:0")
        _check_large(cache, q[rows], [seqs[i] for i in live], [counts[i] for i in live], window=window)


@pytest.mark.parametrize("dim,dtype", [(64, "float32"), (128, "bfloat16"), (192, "float16")])
def test_prefixes_of_very_different_lengths(dim, dtype):
    """Groups whose longest has many times the slots of the others, taken in several rounds."""
    import vicinity_amd as va

    _case(f"{dim} {dtype}")
    prefixes = [299, 4922, 1845, 4029, 391, 4586, 9339, 329]
    cache = share(va.KVCache(80, 8, dim, 1000, code="fp8"))
    k, v = (_rand((sum(prefixes), 8, dim), dtype, i) for i in (1, 2))
    cache.append(k, v, seqs=range(72, 80), counts=prefixes)
    cache.fork([72 + i // 9 for i in range(72)], range(72))
    k, v = (_rand((72 * 19, 8, dim), dtype, i) for i in (3, 4))
    cache.append(k, v, seqs=range(72))
    q = _rand((72, 32, dim), dtype, 5)
    _check_large(cache, q, list(range(72)), [1] * 72)


@pytest.mark.parametrize("forks,empty", [(126, 3), (127, 1), (120, 9), (253, 200)])
def test_launches_of_sequences_without_slots(forks, empty):
    """Beyond the sequences of a launch only empty ones are left."""
    import torch

    import vicinity_amd as va

    cache = share(va.KVCache(forks + empty + 1, 2, 64, forks + 12, block_tokens=64))
    k, v = (_rand((640, 2, 64), "bfloat16", i) for i in (1, 2))
    cache.append(k, v, seqs=[forks + empty])
    cache.fork([forks + empty] * forks, range(forks))
    k, v = (_rand((forks, 2, 64), "bfloat16", i) for i in (3, 4))
    cache.append(k, v, seqs=range(forks))
    n = forks + empty
    q = _rand((n, 8, 64), "bfloat16", 5)
    out, lse = cache.attend(q, seqs=range(n), return_lse=True)
    assert (out[forks:] == 0).all() and torch.isneginf(lse[forks:]).all()
    _check_large(cache, q[:forks], list(range(forks)), [1] * forks)
