"""Attention of sequences that share blocks, which are read once for all of them: against the
definition in 64 bits for each sequence by itself, with the bounds of test_gpu_kv."""

import copy
import random

import numpy as np
import pytest

from test_gpu_kv import OUT_EPS, U, Pair, _check_attend, _rand

pytestmark = pytest.mark.gpu


def _case(msg):
    print(f"[case] kv shared: {msg}", flush=True)


def _torch():
    import torch

    return torch


def share(cache):
    """Shared slots are read once also where that saves little."""
    from vicinity_amd import _lib

    _lib.check(_lib.load().vgpu_test_set_kv_shared_bytes(cache._h, 0))
    return cache


class Forks(Pair):
    def __init__(self, *args, **kw):
        super().__init__(*args, **kw)
        share(self.cache)

    def fork(self, seqs, into, lengths=None):
        self.cache.fork(seqs, into, lengths)
        was = [(copy.deepcopy(self.k[s]), copy.deepcopy(self.v[s])) for s in seqs]
        for i, to in enumerate(into):
            self.k[to], self.v[to] = was[i]
            if lengths is not None:
                for st in was[i]:
                    st.codes, st.scales = st.codes[:lengths[i]], st.scales[:-(-lengths[i] // st.block)]

    def add(self, seqs, counts, dtype="float32", seed=0, gain=1.0):
        t = sum(counts)
        if t:
            self.append(_rand((t, self.heads, self.dim), dtype, seed, gain),
                        _rand((t, self.heads, self.dim), dtype, seed + 1, gain), seqs, counts)


def _family(prefix, own, heads, dim, block, code, dtype="float32", extra=0):
    """Sequence 0 holds the prefix, 1 .. continue it with own[i] tokens of their own."""
    n = len(own)
    blocks = -(-prefix // block) + sum(-(-o // block) + 1 for o in own) + extra
    pair = Forks(n + 1 + (extra > 0), heads, dim, block, code, blocks=blocks)
    pair.add([0], [prefix], dtype, 1)
    pair.fork([0] * n, list(range(1, n + 1)))
    pair.add(list(range(1, n + 1)), own, dtype, 3)
    return pair


def _check_large(cache, q, seqs, counts, window=0, mask=None):
    """The same on the GPU for larger caches: keys and values as read back, each rounded once
    to float32 (u = 2^-24 more of each score's products and of each value)."""
    torch = _torch()
    dim, heads = q.shape[2], cache.num_heads
    group = q.shape[1] // heads
    out, lse = cache.attend(q, seqs=seqs, counts=counts, window=window, mask=mask, return_lse=True)
    scale, at = float(np.float32(1 / np.sqrt(dim))), 0
    for seq, n in zip(seqs, counts):
        got = cache.read(seqs=[seq], fields=("k", "v"))
        k, v = got["k"].double(), got["v"].double()
        slots = len(k)
        last = slots - n + torch.arange(n, device="cuda:0")[:, None]
        slot = torch.arange(slots, device="cuda:0")[None]
        see = (slot <= last) & (slot > last - (window or slots))
        if mask is not None:
            see &= mask[at:at + n, :slots]
        hide = (~see).repeat_interleave(group, dim=0)
        kmax = k.abs().amax(dim=(0, 2))
        for h in range(heads):
            x = q[at:at + n, h * group:h * group + group].double().reshape(n * group, dim)
            s = torch.mm(x, k[:, h].T.contiguous()) * scale
            a = float(scale * x.abs().sum(dim=1).max() * kmax[h])  # not below sum |q k|
            s[hide] = -torch.inf
            wlse = torch.logsumexp(s, dim=1)
            p = torch.exp(s - torch.where(torch.isinf(wlse), 0.0, wlse)[:, None])
            want = torch.mm(p, v[:, h].contiguous())
            e = (dim + 17) * U * (a + 32)
            two = q.dtype == torch.float32
            rel = 2 * e + (2.0 ** -22 if two else 2.0 ** -11) + slots * (2 * U + 2.0 ** -30) + U
            vmax = float(v[:, h].abs().max())
            eps = OUT_EPS[str(q.dtype).split(".")[1]]
            have = out[at:at + n, h * group:h * group + group].double().reshape(n * group, dim)
            assert ((have - want).abs() <= vmax * rel + eps * (want.abs() + vmax * rel)).all(), (seq, h)
            have = lse[at:at + n, h * group:h * group + group].double().reshape(-1)
            seen = ~torch.isinf(wlse)
            assert torch.equal(torch.isneginf(have), ~seen)
            err = (have - wlse)[seen].abs()
            assert (err <= 2 * e + slots * 2 * U + 4 * U * wlse[seen].abs()).all(), (seq, h)
        at += n


def _large(prefix, own, heads, dim, block, code, dtype):
    import vicinity_amd as va

    n = len(own)
    cache = share(va.KVCache(n + 1, heads, dim, -(-prefix // block) + sum(-(-o // block) + 1 for o in own),
                             block_tokens=block, code=code))
    for seqs, counts, seed in (([0], [prefix], 1), (list(range(1, n + 1)), own, 3)):
        if seed > 1:
            cache.fork([0] * n, seqs)
        t = sum(counts)
        cache.append(_rand((t, heads, dim), dtype, seed), _rand((t, heads, dim), dtype, seed + 1), seqs=seqs,
                     counts=counts)
    return cache


def _q(pair, counts, group, dtype, seed=7):
    return _rand((sum(counts), pair.heads * group, pair.dim), dtype, seed)


@pytest.mark.parametrize("code", ["int8", "fp8"])
@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("dim", [1, 64, 80, 128, 192, 250])
def test_types_and_dimensions(code, dtype, dim):
    _case(f"{code} {dtype} dim {dim}")
    pair = _family(333, [1, 40, 7, 100, 64], 2, dim, 32, code)
    seqs = [1, 2, 3, 4, 5]
    _check_attend(pair, _q(pair, [1] * 5, 3, dtype), seqs, [1] * 5)
    _check_attend(pair, _q(pair, [1, 9, 7, 30, 2], 3, dtype), seqs, [1, 9, 7, 30, 2])


@pytest.mark.parametrize("prefix", [256, 257, 287, 288, 300, 319, 320, 513])
@pytest.mark.parametrize("block", [32, 64, 256])
def test_where_the_prefix_ends(prefix, block):
    _case(f"prefix {prefix} block {block}")
    # some have no token of their own, some no whole tile, some many
    pair = _family(prefix, [0, 0, 1, 31, 33, 300, 5], 1, 64, block, "int8")
    seqs = [3, 1, 2, 7, 6, 4, 5, 0]
    _check_attend(pair, _q(pair, [1] * 8, 4, "bfloat16"), seqs, [1] * 8)
    counts = [3, 2, 70, 1, 40, 9, 33, 0]  # more than their own: the queries reach into the prefix
    _check_attend(pair, _q(pair, counts, 4, "bfloat16"), seqs, counts)
    _check_attend(pair, _q(pair, counts, 4, "bfloat16"), seqs, counts, causal=False)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("window", [1, 33, 200, 290, 400, 700, 5000])
def test_windows(dtype, window):
    _case(f"{dtype} window {window}")
    pair = _family(600, [1, 90, 40, 33, 8], 2, 64, 64, "fp8")
    for counts in ([1] * 5, [1, 33, 5, 2, 8]):
        for causal in (True, False):
            _check_attend(pair, _q(pair, counts, 2, dtype), [1, 2, 3, 4, 5], counts, window=window, causal=causal)


@pytest.mark.parametrize("dtype", ["float32", "float16"])
def test_masks(dtype):
    torch = _torch()
    pair = _family(400, [1, 90, 40, 33, 8], 2, 80, 32, "int8")
    seqs, counts = [1, 2, 3, 4, 5], [1, 20, 5, 2, 8]
    q = _q(pair, counts, 2, dtype)
    g = torch.Generator().manual_seed(3)
    mask = torch.rand((36, 500), generator=g) < 0.5
    mask[2] = False  # nothing
    mask[3, :400] = False  # nothing that is shared
    mask[4, 384:] = False  # nothing of its own
    mask[30] = False
    mask = mask.to("cuda:0")
    _check_attend(pair, q, seqs, counts, mask=mask)
    _check_attend(pair, q, seqs, counts, mask=mask.to(torch.uint8) * 7, window=150)
    _check_attend(pair, q, seqs, counts, mask=mask.t().contiguous().t(), causal=False)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("dim,group", [(64, 16), (64, 5), (128, 8), (192, 8), (256, 4)])
def test_many_rows_over_a_long_prefix(dtype, dim, group):
    """Rows enough for the kernel of many rows over the shared slots."""
    _case(f"{dtype} dim {dim} group {group}")
    torch = _torch()
    heads = 16 if dim < 128 else 32  # 98304 tiles of 16 rows
    cache = _large(12000, [1, 70, 33, 5, 200, 64, 1, 2, 3, 4, 5, 6, 7, 8, 9, 10, 40], heads, dim, 128, "int8", "bfloat16")
    seqs = list(range(1, 18))
    q = _rand((17, heads * group, dim), dtype, 7)
    _check_large(cache, q, seqs, [1] * 17)
    _check_large(cache, q, seqs, [1] * 17, window=5000)
    mask = (torch.rand((17, 12200), generator=torch.Generator().manual_seed(1)) < 0.9).to("cuda:0")
    _check_large(cache, q, seqs, [1] * 17, mask=mask)


@pytest.mark.parametrize("dim", [64, 128])
def test_long_queries_over_shared_and_own_slots(dim):
    """Chunks of tokens that continue one document: both kinds of slots by the kernel of many
    rows, or one kind."""
    cache = _large(6000, [300, 1000, 77], 8, dim, 64, "fp8", "bfloat16")
    for counts in ([300, 400, 77], [100, 1, 2], [150, 1000, 77]):
        q = _rand((sum(counts), 32, dim), "bfloat16", 7)
        _check_large(cache, q, [1, 2, 3], counts)
    _check_large(cache, q, [1, 2, 3], counts, window=700)


def test_beams_of_beams():
    """Branches on several levels: of all, of some, of pairs; and sequences that share nothing."""
    pair = Forks(16, 2, 64, 32, "int8", blocks=400)
    pair.add([0, 15], [300, 500], seed=1)
    pair.fork([0, 0, 0], [1, 2, 3])
    pair.add([1, 2, 3], [700, 40, 900], seed=3)
    pair.fork([1, 1, 3, 3, 3, 3], [4, 5, 6, 7, 8, 9])
    pair.add([4, 5, 6, 7, 8, 9], [3, 200, 400, 1, 2, 50], seed=5)
    pair.fork([6, 6], [10, 11])
    pair.add([10, 11, 12], [33, 300, 90], seed=7)
    rng = random.Random(1)
    for _ in range(12):
        seqs = rng.sample(range(16), rng.randint(2, 16))
        counts = [rng.choice([0, 1, 1, 3]) for _ in seqs]
        counts = [min(c, len(pair.k[s].codes)) for s, c in zip(seqs, counts)]
        q = _q(pair, counts, 2, "bfloat16", seed=rng.randrange(1000))
        _check_attend(pair, q, seqs, counts)


@pytest.mark.parametrize("n", [127, 128, 129, 300])
def test_more_sequences_than_one_launch_takes(n):
    _case(f"{n} sequences")
    pair = _family(290, [1 + i % 3 for i in range(n)], 1, 16, 32, "int8")
    seqs = list(range(1, n + 1))
    random.Random(n).shuffle(seqs)
    _check_attend(pair, _q(pair, [1] * n, 2, "float16"), seqs, [1] * n)


def test_many_groups_in_one_call():
    groups, width = 60, 4
    pair = Forks(groups * (width + 1), 1, 16, 32, "fp8", blocks=groups * 20)
    roots = list(range(groups))
    pair.add(roots, [256 + i for i in range(groups)], seed=1)
    kids = list(range(groups, groups * (width + 1)))
    pair.fork([i % groups for i in range(len(kids))], kids)
    pair.add(kids, [1 + i % 40 for i in range(len(kids))], seed=3)
    seqs = kids + roots
    random.Random(5).shuffle(seqs)
    _check_attend(pair, _q(pair, [1] * len(seqs), 2, "bfloat16"), seqs, [1] * len(seqs))


def test_what_is_not_finite_stays_where_it_is_seen():
    torch = _torch()
    nan = float("nan")
    pair = Forks(5, 1, 64, 32, "int8", blocks=100)
    k, v = _rand((320, 1, 64), "float32", 1), _rand((320, 1, 64), "float32", 2)
    v[40, 0, 3] = nan  # one block of the shared slots
    pair.append(k, v, [0], [320])
    pair.fork([0, 0, 0], [1, 2, 3])
    own = _rand((120, 1, 64), "float32", 3)
    own_v = _rand((120, 1, 64), "float32", 4)
    own_v[50] = float("inf")  # the second one's own
    pair.append(own, own_v, [1, 2, 3], [40, 40, 40])
    seqs, counts = [1, 2, 3], [2, 2, 2]
    q = _q(pair, counts, 2, "float32")
    out, lse = pair.cache.attend(q, seqs=seqs, counts=counts, return_lse=True)
    assert torch.isnan(out).all() and torch.isfinite(lse).all()
    # hidden from all: by a mask, then by a window; the second's own is in its third block (20
    # of its own are before it)
    mask = torch.ones((6, 400), dtype=torch.bool, device="cuda:0")
    mask[:, 32:64] = False
    out = pair.cache.attend(q, seqs=seqs, counts=counts, mask=mask)
    assert torch.isfinite(out[[0, 1, 4, 5]]).all() and torch.isnan(out[2:4]).all()
    mask[2:4, 320:352] = False
    out = pair.cache.attend(q, seqs=seqs, counts=counts, mask=mask)
    assert torch.isfinite(out).all()
    out = pair.cache.attend(q, seqs=seqs, counts=counts, window=290)
    assert torch.isfinite(out[[0, 1, 4, 5]]).all() and torch.isnan(out[2:4]).all()
    # a query that is not finite is NaN by itself
    q[3, 1, 7] = float("inf")
    out, lse = pair.cache.attend(q, seqs=seqs, counts=counts, mask=mask, return_lse=True)
    bad = torch.zeros((6, 2), dtype=torch.bool, device="cuda:0")
    bad[3, 1] = True
    assert torch.equal(torch.isnan(out).any(dim=2), bad) and torch.equal(torch.isnan(lse), bad)
    # and 0 where it sees nothing
    mask[3] = False
    out, lse = pair.cache.attend(q, seqs=seqs, counts=counts, mask=mask, return_lse=True)
    assert torch.isfinite(out).all() and (out[3] == 0).all() and torch.isneginf(lse[3]).all()


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_scales_of_any_size(dtype):
    """Values of shared and own slots that lie far apart."""
    for prefix_gain, own_gain in ((2.0 ** 40, 1.0), (1.0, 2.0 ** 40), (2.0 ** -60, 2.0 ** -60), (0.0, 1.0), (1.0, 0.0)):
        pair = Forks(4, 1, 64, 32, "int8", blocks=100)
        for seqs, counts, gain, seed in (([0], [400], prefix_gain, 1), ([1, 2, 3], [40, 1, 90], own_gain, 5)):
            if seqs != [0]:
                pair.fork([0] * 3, seqs)
            t = sum(counts)
            pair.append(_rand((t, 1, 64), "float32", seed), _rand((t, 1, 64), "float32", seed + 1) * gain, seqs, counts)
        counts = [2, 1, 5]
        _check_attend(pair, _q(pair, counts, 2, dtype), [1, 2, 3], counts)


def test_strides_outputs_and_streams():
    torch = _torch()
    pair = _family(500, [30, 40, 50], 2, 64, 64, "int8")
    counts = [2, 3, 4]
    big = _rand((9, 12, 128), "bfloat16", 5)
    for q in (big[:, 2:10, ::2], big[:, :8, 32:96], big.flip(0)[:, 4:, 64:]):
        _check_attend(pair, q, [1, 2, 3], counts)
    q = big[:, :8, :64].contiguous()
    want = pair.cache.attend(q, seqs=[1, 2, 3], counts=counts)
    out = torch.empty_like(want)
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for i in range(6):
        pair.cache.attend(q, seqs=[1, 2, 3], counts=counts, out=out, stream=streams[i % 2])
        torch.cuda.synchronize()
        assert torch.equal(out, want)
    # rows of other sequences are left alone
    want = pair.cache.attend(q[2:5], seqs=[2], counts=[3])
    out.fill_(7.0)
    pair.cache.attend(q[2:5], seqs=[2], counts=[3], out=out[2:5])
    assert torch.equal(out[2:5], want) and (out[:2] == 7.0).all() and (out[5:] == 7.0).all()
    want = pair.cache.attend(q[2:], seqs=[2, 3], counts=counts[1:])
    pair.cache.attend(q[2:], seqs=[2, 3], counts=counts[1:], out=out[2:])
    assert torch.equal(out[2:], want) and (out[:2] == 7.0).all()


@pytest.mark.parametrize("seed", range(8))
def test_random_families(seed):
    rng = random.Random(seed)
    heads, dim, block = rng.choice([1, 2, 5]), rng.choice([16, 64, 96, 128]), rng.choice([32, 64, 128])
    n, group = rng.randint(2, 12), rng.choice([1, 2, 4, 7])
    dtype, code = rng.choice(["float32", "float16", "bfloat16"]), rng.choice(["int8", "fp8"])
    prefix, own = rng.randint(200, 3000), [rng.choice([0, 1, 20, 64, 333]) for _ in range(n)]
    _case(f"{seed}: heads {heads} dim {dim} block {block} {dtype} {code} prefix {prefix} own {own}")
    pair = _family(prefix, own, heads, dim, block, code)
    seqs = list(range(n + 1))
    rng.shuffle(seqs)
    counts = [rng.choice([0, 1, 2, 17, 60]) for _ in seqs]
    _check_attend(pair, _q(pair, counts, group, dtype), seqs, counts, causal=rng.random() < 0.8,
                  window=rng.choice([0, 0, 300, 1000]))
