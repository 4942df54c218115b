"""How attention of few rows is split over workgroups: no workgroup may be left with a large
part of the work that all of them have."""

import ctypes
import random

import numpy as np
import pytest

TILE, ROWS, PLACES = 32, 16, 768  # slots of a tile, rows of a workgroup, workgroups at once


def _splits(lens, counts, heads, group):
    from vicinity_amd import _lib

    n = len(lens)
    a, b = np.array(lens, np.int64), np.array(counts, np.int64)
    splits, tiles = np.zeros(n, np.int32), np.zeros(n, np.int32)
    p = [x.ctypes.data_as(ctypes.c_void_p) for x in (a, b, splits, tiles)]
    _lib.check(_lib.load().vgpu_test_host_kv_splits(p[0], p[1], n, heads, group, p[2], p[3]))
    return splits, tiles


def _check(lens, counts, heads, group):
    splits, tiles = _splits(lens, counts, heads, group)
    all_tiles = (np.array(lens) + TILE - 1) // TILE
    row_tiles = (np.array(counts) * group + ROWS - 1) // ROWS
    assert (splits >= 1).all() and (tiles >= 1).all()
    assert (splits * tiles >= all_tiles).all()            # all tiles are gone over
    assert ((splits - 1) * tiles < np.maximum(all_tiles, 1)).all()  # and no split is without
    share = (row_tiles * heads * all_tiles).sum() / PLACES
    busy = (row_tiles > 0) & (all_tiles > 0)
    assert (tiles[busy] <= max(2.5 * share, 16)).all(), (tiles[busy].max(), share)
    # partial results for no more than the splits that the work asks for
    assert (row_tiles * heads * (splits - 1)).sum() <= 2 * PLACES


@pytest.mark.parametrize("shorts,heads,group,count", [
    (127, 8, 4, 1), (108, 8, 4, 1), (99, 8, 1, 1), (60, 8, 4, 1), (27, 32, 4, 1), (63, 12, 16, 2), (1, 8, 8, 1)])
@pytest.mark.parametrize("longest", [2048, 131_072, 1 << 22])
def test_one_long_sequence_among_short_ones(shorts, heads, group, count, longest):
    lens = [100 + i % 7 for i in range(shorts)]
    lens.insert(shorts // 2, longest)
    _check(lens, [count] * len(lens), heads, group)


@pytest.mark.parametrize("seed", range(200))
def test_any_batch(seed):
    rng = random.Random(seed)
    n = rng.randint(1, 128)
    lens = [int(2 ** rng.uniform(0, 17)) for _ in range(n)]
    counts = [rng.choice([0, 1, 1, 1, 5]) for _ in range(n)]
    _check(lens, counts, rng.choice([1, 2, 8, 8, 12, 32, 64]), rng.choice([1, 4, 8]))
