"""Sequences of a KVCache that continue one another: fork, copies, compaction, and what
append, truncate, evict and attend do to blocks that several sequences hold.  Every sequence
has to hold, bit for bit, what it would hold alone."""

import copy
import random

import numpy as np
import pytest

import kv_reference as ref

pytestmark = pytest.mark.gpu


def _case(msg):
    print(f"[case] kv fork: {msg}", flush=True)


def _torch():
    import torch

    return torch


def _np(t):
    return t.detach().float().cpu().numpy()


class Alone:
    """One sequence by itself."""

    def __init__(self, heads, dim, block, code):
        self.k, self.v = ref.Store(heads, dim, block, code), ref.Store(heads, dim, block, code)
        self.positions = np.zeros((0, heads), np.int32)
        self.weights = np.zeros((0, heads), np.float32)
        self.next, self.block = 0, block

    def __len__(self):
        return len(self.positions)

    def append(self, k, v, weights):
        n, h = k.shape[:2]
        self.k.append(k)
        self.v.append(v)
        new = np.arange(self.next, self.next + n, dtype=np.int32)
        self.positions = np.concatenate([self.positions, np.repeat(new[:, None], h, axis=1)])
        self.weights = np.concatenate([self.weights, weights])
        self.next += n

    def cut(self, n):
        self.next = self.next - (len(self) - n) if n else 0
        for st in (self.k, self.v):
            st.codes, st.scales = st.codes[:n], st.scales[:-(-n // self.block)]
        self.positions, self.weights = self.positions[:n], self.weights[:n]

    def evict(self, budget, recent):
        if len(self) <= budget:
            return
        stay, _ = ref.keep_slots(self.weights, budget, recent)
        heads = np.arange(self.weights.shape[1])[None]
        self.k, self.v = self.k.kept(stay), self.v.kept(stay)
        self.positions, self.weights = self.positions[stay, heads], self.weights[stay, heads]


class Both:
    """A cache and its sequences, each alone."""

    def __init__(self, seqs, heads=2, dim=40, block=32, code="int8", blocks=64, **kw):
        import vicinity_amd as va

        self.cache = va.KVCache(seqs, heads, dim, blocks, block_tokens=block, code=code, **kw)
        self.seqs = [Alone(heads, dim, block, code) for _ in range(seqs)]
        self.heads, self.dim, self.seed = heads, dim, 0

    def append(self, seqs, counts, gain=1.0, stream=None):
        torch = _torch()
        t = sum(counts)
        self.seed += 1
        g = torch.Generator().manual_seed(self.seed)
        k = torch.randn((t, self.heads, self.dim), generator=g) * gain
        v = torch.randn((t, self.heads, self.dim), generator=g) * gain
        w = torch.rand((t, self.heads), generator=g)
        dev = [x.to("cuda:0") for x in (k, v, w)]
        torch.cuda.synchronize()
        self.cache.append(dev[0], dev[1], seqs=seqs, counts=counts, weights=dev[2], stream=stream)
        at = 0
        for s, n in zip(seqs, counts):
            self.seqs[s].append(k[at:at + n].numpy(), v[at:at + n].numpy(), w[at:at + n].numpy())
            at += n

    def fork(self, seqs, into, lengths=None, **kw):
        self.cache.fork(seqs, into, lengths, **kw)
        was = [copy.deepcopy(self.seqs[s]) for s in seqs]
        for i, (s, to) in enumerate(zip(was, into)):
            if lengths is not None and lengths[i] < len(s):
                s.cut(lengths[i])
            self.seqs[to] = s

    def truncate(self, lengths, seqs):
        self.cache.truncate(lengths, seqs=seqs)
        for s, n in zip(seqs, lengths):
            self.seqs[s].cut(n)

    def evict(self, budget, recent, seqs):
        self.cache.evict(budget, recent, seqs=seqs)
        for s in seqs:
            self.seqs[s].evict(budget, recent)

    def check(self):
        assert self.cache.lengths.tolist() == [len(s) for s in self.seqs]
        got = self.cache.read()
        for name, want in (("k", [s.k.values32() for s in self.seqs]), ("v", [s.v.values32() for s in self.seqs]),
                           ("positions", [s.positions for s in self.seqs]),
                           ("weights", [s.weights for s in self.seqs])):
            have = got[name].cpu().numpy()
            assert np.array_equal(have, np.concatenate(want), equal_nan=True), name


@pytest.mark.parametrize("copied", [False, True])
@pytest.mark.parametrize("code", ["int8", "fp8"])
@pytest.mark.parametrize("length", [1, 31, 32, 33, 64, 95])
def test_children_go_their_own_ways(copied, code, length):
    _case(f"copied {copied} {code} length {length}")
    b = Both(5, code=code)
    b.append([0], [length])
    free = b.cache.info()["free_blocks"]
    b.fork([0, 0, 0], [1, 2, 3], copy=copied)
    assert b.cache.info()["free_blocks"] == free - (3 * -(-length // 32) if copied else 0)
    b.check()
    for step in range(3):  # larger tokens each time, so that scales of begun blocks grow
        b.append([1, 0, 3], [1, 2, 40], gain=1.0 + step)
        b.check()
    b.append([2], [1], gain=0.1)
    b.check()
    b.truncate([0, 0, 0, 0], [0, 1, 2, 3])
    assert b.cache.info()["free_blocks"] == 64
    b.check()


def test_the_last_holder_keeps_its_block():
    b = Both(3, blocks=4)
    b.append([0], [40])
    b.fork([0], [1])
    assert b.cache.info()["free_blocks"] == 2
    b.append([0, 1], [1, 1])  # one of them copies the begun block, the other keeps it
    assert b.cache.info()["free_blocks"] == 1
    b.check()
    b.fork([1], [2])
    b.truncate([0], [1])
    b.append([2], [1])  # nobody else holds it now
    assert b.cache.info()["free_blocks"] == 1
    b.check()


@pytest.mark.parametrize("blocks_each", [3, 70])  # entries by kernel arguments, or copied rows
def test_beams_are_reordered(blocks_each):
    _case(f"reorder, {blocks_each} blocks each")
    n = 6
    b = Both(n, heads=1, dim=8, blocks=n * (blocks_each + 6))
    b.append(list(range(n)), [32 * blocks_each - 5 * i for i in range(n)])
    b.check()
    for parents in ([1, 0, 2, 3, 4, 5], [5, 5, 5, 0, 1, 2], [0, 0, 3, 3, 4, 4], [1, 2, 3, 4, 5, 0]):
        b.fork(parents, list(range(n)))
        b.check()
        b.append(list(range(n)), [1, 2, 3, 30, 31, 32])
        b.check()
    b.truncate([0] * n, list(range(n)))
    assert b.cache.info()["free_blocks"] == n * (blocks_each + 6)


@pytest.mark.parametrize("copied", [False, True])
def test_lengths_and_forks_of_oneself(copied):
    b = Both(4, blocks=40)
    b.append([0, 1], [70, 5])
    b.fork([0, 0, 1, 0], [0, 1, 2, 3], [33, 64, 0, 70], copy=copied)
    b.check()
    b.append([0, 1, 2, 3], [3, 3, 3, 3])
    b.check()
    b.fork([], [])
    b.check()


def test_many_sequences_in_one_call():
    n = 200  # more than one launch's
    b = Both(n + 1, heads=1, dim=4, blocks=n + 80)
    b.append([n], [66 * 32 + 1])
    b.fork([n] * n, list(range(n)))
    b.append(list(range(n)), [1] * n)
    b.check()
    order = list(range(n))
    random.Random(3).shuffle(order)
    b.fork(order, list(range(n)))
    b.check()


def test_evicting_forks():
    b = Both(4, blocks=12)
    b.append([0], [150])  # 5 blocks
    b.fork([0, 0], [1, 2])
    b.append([1], [20])
    b.check()
    # 12 blocks, 7 in use: 0, 1 and 2 each take 2 anew, and what they let go comes back only
    # when its last holder has gone
    b.evict(64, 10, [0, 1, 2])
    b.check()
    assert b.cache.info()["free_blocks"] == 6
    b.append([0, 1, 2, 3], [1, 40, 1, 1])
    b.check()


def test_eviction_counts_what_comes_back():
    b = Both(4, blocks=8)
    b.append([0], [160])  # 5 blocks, 3 free
    b.fork([0, 0, 0], [1, 2, 3])
    free = b.cache.info()["free_blocks"]
    with pytest.raises(RuntimeError, match="free blocks"):
        b.cache.evict(64, 0, seqs=[0, 1, 2])  # the fourth still holds the five
    assert b.cache.info()["free_blocks"] == free
    b.check()
    b.evict(64, 0, [0])
    b.check()
    with pytest.raises(RuntimeError, match="free blocks"):
        b.cache.evict(64, 0, seqs=[1, 2, 3])
    b.evict(32, 0, [1])
    b.truncate([0], [2])
    b.check()
    assert b.cache.info()["free_blocks"] == 0
    b.truncate([0], [1])
    b.evict(32, 0, [3])
    b.check()


def test_positions_go_on_as_the_parents():
    b = Both(4, blocks=30)
    b.append([0, 1], [50, 40])
    b.evict(0, 0, [0])  # nothing is left, and the next token has position 50
    b.evict(10, 2, [1])
    b.fork([0, 1, 1], [2, 3, 1], [0, 10, 7])
    b.append([0, 1, 2, 3], [2, 2, 2, 2])
    b.check()
    assert b.seqs[2].positions[0, 0] == 50 and b.seqs[3].positions[-1, 0] == 41


@pytest.mark.parametrize("num_blocks", [None, 24, 40, 64])
def test_compaction(num_blocks):
    _case(f"compact to {num_blocks}")
    b = Both(6, blocks=40)
    for step in range(4):  # blocks of the sequences in turn
        b.append([0, 1, 2, 3], [40, 33, 1, 64])
    b.fork([1], [4])
    b.fork([3], [5], [70])
    b.truncate([10, 0, 0, 64], [0, 1, 2, 3])
    b.check()
    used = 40 - b.cache.info()["free_blocks"]
    moved = b.cache.compact(num_blocks)
    total = num_blocks or 40
    assert moved == used if total != 40 else 0 < moved < used
    assert b.cache.num_blocks == total and b.cache.info()["free_blocks"] == total - used
    b.check()
    if num_blocks in (None, 40):
        assert b.cache.compact(num_blocks) == 0
    b.append([0, 4, 5, 1], [40, 1, 3, 5])
    b.check()
    with pytest.raises(ValueError, match="more than num_blocks"):
        b.cache.compact(3)
    b.check()
    b.truncate([0] * 6, list(range(6)))
    assert b.cache.info()["free_blocks"] == total
    b.cache.compact(1)
    b.append([3], [32])
    b.check()
    with pytest.raises(RuntimeError, match="more blocks"):
        b.append([3], [1])


def test_compaction_of_many_gaps():
    n = 500  # more runs than one launch takes, and rows of many columns
    b = Both(3, heads=1, dim=4, blocks=2 * n + 5)
    for _ in range(n):  # blocks of the two in turn
        b.append([0, 1], [32, 32])
    b.fork([1], [2])
    b.truncate([0], [0])
    b.append([2], [70])
    b.check()
    assert b.cache.compact() > n // 3
    b.check()
    assert b.cache.compact(n + 10) == n + 3
    b.check()


@pytest.mark.parametrize("seed", range(6))
def test_random_walks(seed):
    rng = random.Random(seed)
    heads, dim, block = rng.choice([(1, 8, 32), (3, 40, 64), (2, 72, 32)])
    code = rng.choice(["int8", "fp8"])
    _case(f"walk {seed}: heads {heads} dim {dim} block {block} {code}")
    n = 5
    b = Both(n, heads, dim, block, code, blocks=48)
    for step in range(40):
        what = rng.choice(["append", "append", "append", "fork", "fork", "copy", "truncate", "evict", "compact"])
        ids = rng.sample(range(n), rng.randint(1, n))
        try:
            if what == "append":
                b.append(ids, [rng.choice([0, 1, 1, 5, 40, 70]) for _ in ids], gain=rng.choice([0.5, 1.0, 2.0]))
            elif what in ("fork", "copy"):
                src = [rng.randrange(n) for _ in ids]
                lens = None if rng.random() < 0.5 else [rng.randint(0, len(b.seqs[s])) for s in src]
                b.fork(src, ids, lens, copy=what == "copy")
            elif what == "truncate":
                b.truncate([rng.choice([0, len(b.seqs[s]) // 2, len(b.seqs[s])]) for s in ids], ids)
            elif what == "evict":
                b.evict(rng.choice([40, 64, 100]), rng.choice([0, 10]), ids)
            else:
                b.cache.compact(rng.choice([None, None, 48, 56]))
        except (RuntimeError, ValueError) as e:
            # the pool is full, or smaller: nothing has changed (append: nor the model)
            assert "block" in str(e)
            if what == "append":
                b.truncate([0] * n, list(range(n)))
        b.check()


def _attend(cache, q, seqs, counts, **kw):
    out, lse = cache.attend(q, seqs=seqs, counts=counts, return_lse=True, **kw)
    return [out, lse, cache.read(seqs=seqs, fields=("weights",))["weights"]]


@pytest.mark.parametrize("queries", [1, 60])  # kept scores, or a second pass
def test_accumulated_weights_are_each_sequences_own(queries):
    torch = _torch()
    import vicinity_amd as va

    caches = []
    for copied in (False, True):
        g = torch.Generator().manual_seed(5)
        cache = va.KVCache(5, 2, 64, 60, block_tokens=32)
        k, v, k2, v2 = (torch.randn((t, 2, 64), generator=g).to("cuda:0") for t in (150, 150, 180, 180))
        cache.append(k, v, seqs=[0], counts=[150])
        cache.fork([0, 0, 0], [1, 2, 3], copy=copied)
        cache.append(k2, v2, seqs=[0, 1, 2], counts=[60, 60, 60])
        caches.append(cache)
    g = torch.Generator().manual_seed(6)
    for decay in (0.0, 1.0, 0.5):
        q = torch.randn((2 * queries, 4, 64), generator=g).to("cuda:0", torch.bfloat16)
        got = [_attend(c, q, [1, 2], [queries, queries], decay=decay) for c in caches]
        for a, b in zip(*got):
            assert torch.equal(a, b)
        # those that took no part keep theirs
        rest = [c.read(seqs=[0, 3], fields=("weights",))["weights"] for c in caches]
        assert torch.equal(*rest) and not rest[0].any()


def test_weights_of_shared_blocks_need_room():
    torch = _torch()
    b = Both(3, heads=1, dim=64, blocks=5)
    b.append([0], [96])
    b.fork([0], [1])
    q = torch.ones((1, 1, 64), device="cuda:0")
    with pytest.raises(RuntimeError, match="weights of shared blocks") as e:
        b.cache.attend(q, seqs=[1], counts=[1], decay=1.0)
    from vicinity_amd import _lib

    assert e.value.code == _lib.ERR_OUT_OF_MEMORY
    b.check()
    b.cache.attend(q, seqs=[1], counts=[1])  # without weights nothing is copied
    assert b.cache.info()["free_blocks"] == 2
    b.check()


def test_refusals_change_nothing():
    torch = _torch()
    b = Both(4, blocks=5)
    b.append([0], [100])
    b.fork([0], [1])
    free = b.cache.info()["free_blocks"]
    for call, error, match in [
            (lambda: b.cache.fork([0, 0], [2, 3], copy=True), RuntimeError, "free blocks"),
            (lambda: b.cache.fork([0], [4]), ValueError, "out of range"),
            (lambda: b.cache.fork([4], [0]), ValueError, "out of range"),
            (lambda: b.cache.fork([-1], [0]), ValueError, "out of range"),
            (lambda: b.cache.fork([0, 0], [2, 2]), ValueError, "twice"),
            (lambda: b.cache.fork([0], [2, 3]), ValueError, "into names"),
            (lambda: b.cache.fork([0], [2], [101]), ValueError, "outside sequence"),
            (lambda: b.cache.fork([0], [2], [-1]), ValueError, "outside sequence"),
            (lambda: b.cache.fork([0], [2], [1, 2]), ValueError, "one entry"),
            (lambda: b.cache.fork([0.5], [2]), ValueError, "integers"),
            (lambda: b.cache.compact(0), ValueError, "num_blocks"),
            (lambda: b.cache.compact(1.5), ValueError, "num_blocks"),
            (lambda: b.cache.compact(3), ValueError, "num_blocks"),
            (lambda: b.append([0, 1], [1, 40]), RuntimeError, "more blocks")]:
        with pytest.raises(error, match=match):
            call()
        assert b.cache.info()["free_blocks"] == free
        b.check()
    b.append([1], [1])  # takes the last block
    with pytest.raises(RuntimeError, match="more blocks"):
        b.fork([0], [2])
        b.append([2], [1])
    b.check()
    g = torch.cuda.CUDAGraph()
    x = torch.zeros(1, device="cuda:0")
    with torch.cuda.graph(g):
        x.add_(1)
        for call in (lambda: b.cache.fork([0], [3]), lambda: b.cache.compact()):
            with pytest.raises(ValueError, match="captured"):
                call()
    b.check()


def test_streams_of_their_own():
    torch = _torch()
    b = Both(5, heads=4, dim=64, blocks=400)
    streams = [torch.cuda.Stream() for _ in range(3)]
    b.append([0], [700])
    for i in range(12):
        b.fork([0, 0, 1], [1, 2, 3], stream=streams[i % 3])
        b.append([1, 2, 0], [1, 33, 2], stream=streams[(i + 1) % 3])
        if i % 4 == 3:
            b.cache.compact(stream=streams[(i + 2) % 3])
    b.check()


def test_blocks_past_32_bits():
    """Copies at byte offsets past 2^32."""
    torch = _torch()
    import vicinity_amd as va

    heads, dim, block = 64, 256, 256  # 8 MiB a block
    cache = va.KVCache(3, heads, dim, 600, block_tokens=block)
    k = torch.randn((block, heads, dim), device="cuda:0")
    for _ in range(270):
        cache.append(k, k, seqs=[0], counts=[block])
    cache.append(k, -k, seqs=[1], counts=[block])
    cache.fork([0, 1], [1, 2], [0, block], copy=True)
    cache.fork([2], [1], copy=True)  # blocks around number 270
    want = cache.read(seqs=[2], fields=("k", "v", "positions"))
    cache.truncate([0], seqs=[0])
    assert cache.compact() == 2
    for seq in (1, 2):
        got = cache.read(seqs=[seq], fields=("k", "v", "positions"))
        assert all(torch.equal(got[f], want[f]) for f in want)
    assert cache.compact(8) == 2
    got = cache.read(seqs=[1], fields=("k", "v", "positions"))
    assert all(torch.equal(got[f], want[f]) for f in want)


def test_two_threads_fork_one_cache():
    """Threads on streams of their own, each with its own sequences of one cache."""
    import threading

    torch = _torch()
    b = Both(10, heads=2, dim=64, blocks=300)
    b.append([0, 5], [333, 402])
    torch.cuda.synchronize()
    plan = {first: [([first + i for i in order], [1 + (i * 7 + first) % 40 for i in range(5)])
                    for order in ([0, 0, 0, 0, 0], [3, 1, 4, 1, 0], [2, 2, 0, 4, 3], [1, 0, 3, 2, 4])]
            for first in (0, 5)}
    tokens = {}
    for first, steps in plan.items():
        for s, (_, counts) in enumerate(steps):
            g = torch.Generator().manual_seed(100 * first + s)
            t = sum(counts)
            tokens[first, s] = (torch.randn((t, 2, 64), generator=g), torch.randn((t, 2, 64), generator=g),
                                torch.rand((t, 2), generator=g))
    dev = {key: [x.to("cuda:0") for x in v] for key, v in tokens.items()}
    torch.cuda.synchronize()
    failed = []

    def work(first):
        try:
            stream = torch.cuda.Stream()
            own = list(range(first, first + 5))
            for s, (parents, counts) in enumerate(plan[first]):
                k, v, w = dev[first, s]
                b.cache.fork(parents, own, stream=stream)
                b.cache.append(k, v, seqs=own, counts=counts, weights=w, stream=stream)
        except Exception as e:  # noqa: BLE001
            failed.append(e)

    threads = [threading.Thread(target=work, args=(first,)) for first in plan]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed
    torch.cuda.synchronize()
    for first, steps in plan.items():
        for s, (parents, counts) in enumerate(steps):
            was = [copy.deepcopy(b.seqs[p]) for p in parents]
            at = 0
            for i, n in enumerate(counts):
                k, v, w = (x[at:at + n].numpy() for x in tokens[first, s])
                was[i].append(k, v, w)
                b.seqs[first + i] = was[i]
                at += n
    b.check()
