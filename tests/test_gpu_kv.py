"""The attention memory (KVCache) on the GPU against its definitions in 64 bits.

Stored values are the format's and have to be equal bit for bit.  Attention has the
bounds below, from the arithmetic: u = 2^-24 is float32's rounding.
  scores   a sum of D exact products in float32, then a few scalings and the exponential:
           e = (D + 16) u (A + 32) relative in every p, A the largest scale * sum |q k|
  p        rounded to half precision (unit roundoff 2^-11) for 16-bit queries, to two
           halves (2^-22) for float32 ones; what is below 2^-30 of the largest may be
           lost, n such slots
  sums     n u
  output   rounded to its type: unit roundoff 2^-8 bfloat16, 2^-11 float16, 2^-24 float32
"""

import numpy as np
import pytest

import kv_reference as ref

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
OUT_EPS = {"bfloat16": 2.0 ** -8, "float16": 2.0 ** -11, "float32": 2.0 ** -24}


def _case(msg):
    print(f"[case] kv: {msg}", flush=True)


def _torch():
    import torch

    return torch


def _rand(shape, dtype, seed, gain=1.0):
    torch = _torch()
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(shape, generator=g) * gain
    if len(shape) == 3 and shape[2] > 2:
        x[:, :, ::3] *= 3.0
    return x.to(getattr(torch, dtype)).to("cuda:0")


def _np(t):
    return t.detach().float().cpu().numpy()


class Pair:
    """A KVCache and its reference, fed with the same tokens."""

    def __init__(self, seqs, heads, dim, block, code, blocks=None):
        import vicinity_amd as va

        self.heads, self.dim, self.block, self.code = heads, dim, block, code
        self.cache = va.KVCache(seqs, heads, dim, blocks or 64, block_tokens=block, code=code)
        self.k = [ref.Store(heads, dim, block, code) for _ in range(seqs)]
        self.v = [ref.Store(heads, dim, block, code) for _ in range(seqs)]

    def append(self, k, v, seqs, counts, **kw):
        self.cache.append(k, v, seqs=seqs, counts=counts, **kw)
        at = 0
        for s, n in zip(seqs, counts):
            self.k[s].append(_np(k[at:at + n]))
            self.v[s].append(_np(v[at:at + n]))
            at += n

    def check_values(self, seqs=None):
        seqs = range(len(self.k)) if seqs is None else seqs
        got = self.cache.read(seqs=list(seqs))
        for name, stores in (("k", self.k), ("v", self.v)):
            want = np.concatenate([stores[s].values32() for s in seqs])
            assert np.array_equal(_np(got[name]), want, equal_nan=True), name
        return got


def _check_attend(pair, q, seqs, counts, *, scale=None, causal=True, window=0, mask=None,
                  decay=None):
    torch = _torch()
    dtype = str(q.dtype).split(".")[1]
    before = [_np(pair.cache.read(seqs=[s], fields=("weights",))["weights"]) for s in seqs]
    out, lse = pair.cache.attend(q, seqs=seqs, counts=counts, scale=scale, causal=causal,
                                 window=window, mask=mask, decay=decay, return_lse=True)
    assert out.dtype == q.dtype and out.shape == q.shape and lse.dtype == torch.float32
    scale = 1 / np.sqrt(pair.dim) if scale is None else scale
    # the kernel takes the scale in float32
    scale = float(np.float32(scale))
    at = 0
    for s, n, w0 in zip(seqs, counts, before):
        k, v = pair.k[s].values(), pair.v[s].values()
        see = ref.visible(len(k), n, causal, window)
        if mask is not None:
            see &= mask[at:at + n, :len(k)].cpu().numpy().astype(bool)
        qs = _np(q[at:at + n]).astype(np.float64)
        want, wlse, w = ref.attend(qs, k, v, see, scale)
        g = q.shape[1] // pair.heads
        a, vmax = 0.0, 0.0
        if len(k) and n:
            kk = np.repeat(np.abs(np.nan_to_num(k)), g, axis=1)
            a = scale * np.einsum("thd,nhd->thn", np.abs(qs), kk).max()
            vmax = np.nanmax(np.abs(v))
        e = (pair.dim + 16) * U * (abs(a) + 32)
        p_eps = 2.0 ** -22 if dtype == "float32" else 2.0 ** -11
        rel = 2 * e + p_eps + len(k) * (2 * U + 2.0 ** -30)
        got = _np(out[at:at + n]).astype(np.float64)
        err = np.abs(got - want)
        limit = vmax * rel + OUT_EPS[dtype] * (np.abs(want) + vmax * rel)
        assert (err <= limit).all(), (s, float((err - limit).max()), float(err.max()))
        gl = _np(lse[at:at + n]).astype(np.float64)
        empty = np.isneginf(wlse)
        assert np.array_equal(np.isneginf(gl), empty)
        lerr = np.abs(gl[~empty] - wlse[~empty])
        assert (lerr <= 2 * e + len(k) * 2 * U + 4 * U * np.abs(wlse[~empty])).all()
        assert (got[empty] == 0).all()
        after = _np(pair.cache.read(seqs=[s], fields=("weights",))["weights"])
        if decay is None:
            assert np.array_equal(after, w0, equal_nan=True)
        else:
            total = decay * w0.astype(np.float64) + w
            rows = n * g
            tol = (3 * e + (len(k) + rows + 8) * 2 * U) * total + rows * 2.0 ** -100
            assert (np.abs(after - total) <= tol).all()
        at += n


# ---- append and read ----------------------------------------------------------


@pytest.mark.parametrize("code", ["int8", "fp8"])
@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("heads,dim,block", [(1, 1, 32), (3, 40, 32), (2, 64, 64), (2, 80, 128),
                                             (1, 128, 256), (2, 192, 64), (1, 250, 32)])
def test_append_in_pieces_equals_the_format(code, dtype, heads, dim, block):
    _case(f"append {code} {dtype} heads {heads} dim {dim} block {block}")
    pair = Pair(3, heads, dim, block, code)
    for step, counts in enumerate([[1, 0, 33], [31, 5, 1], [1, 70, 2], [0, 1, 1], [90, 1, 64]]):
        t = sum(counts)
        # later pieces are larger, so that the scales of begun blocks grow
        k = _rand((t, heads, dim), dtype, 10 * step, 1.0 + 0.5 * step)
        v = _rand((t, heads, dim), dtype, 10 * step + 1, 1.0 + 0.3 * step)
        pair.append(k, v, [0, 1, 2], counts)
    got = pair.check_values()
    lens = pair.cache.lengths
    assert list(lens) == [123, 77, 101]
    pos = np.concatenate([np.arange(n) for n in lens])
    assert np.array_equal(got["positions"].cpu().numpy(), np.tile(pos[:, None], (1, heads)))
    assert not got["weights"].any()


@pytest.mark.parametrize("code", ["int8", "fp8"])
def test_every_half_precision_number_is_rounded_like_the_format(code):
    """All finite float16 values, a scale of 1 (the block's largest is Z)."""
    torch = _torch()
    _case(f"append {code}: every float16 within the code's range")
    z = float(ref.Z[code])
    x = torch.arange(-32768, 32768, dtype=torch.int32).to(torch.int16).view(torch.float16)
    x = x[torch.isfinite(x) & (x.abs() <= z)]
    # 255 of them and Z in every block of 256 slots
    pad = -len(x) % 255
    x = torch.cat([x, x.new_zeros(pad)]).view(-1, 255)
    x = torch.cat([x, x.new_full((len(x), 1), z)], dim=1).reshape(-1, 1, 1).to("cuda:0")
    pair = Pair(1, 1, 1, 256, code, blocks=len(x) // 256)
    pair.append(x, -x, [0], [len(x)])
    pair.check_values()


def test_strides_and_alignment():
    torch = _torch()
    _case("append and attend: heads first, sliced, reversed roles, one dim apart, misaligned")
    heads, dim, t = 3, 64, 45
    base = _rand((heads, t, dim), "bfloat16", 1)
    wide = _rand((t, heads, 2 * dim + 8), "bfloat16", 2)
    forms = [base.transpose(0, 1), wide[:, :, 3:3 + dim], wide[:, :, :2 * dim:2],
             wide[:, :, 8:8 + dim], base[0][:, None, :].expand(t, heads, dim),
             _rand((t, dim, heads), "float32", 3).transpose(1, 2),
             _rand((1, heads, dim), "float16", 4).expand(t, heads, dim)]
    for i, x in enumerate(forms):
        pair = Pair(1, heads, dim, 32, "int8")
        pair.append(x, x.flip(0), [0], [t])
        pair.check_values()
        _check_attend(pair, x[-2:], [0], [2])


def test_given_positions_and_weights_are_kept():
    torch = _torch()
    _case("append with positions and weights")
    import vicinity_amd as va

    cache = va.KVCache(2, 2, 64, 8, block_tokens=32)
    k = _rand((40, 2, 64), "bfloat16", 5)
    pos = torch.randint(0, 10_000, (40, 2), dtype=torch.int32).to("cuda:0")
    wts = torch.rand((40, 2)).to("cuda:0")
    cache.append(k, k, counts=[33, 7], positions=pos, weights=wts)
    got = cache.read()
    assert torch.equal(got["positions"], pos) and torch.equal(got["weights"], wts)
    # counted on from the tokens appended, less those taken back
    cache.truncate([30, 7])
    cache.append(k[:2], k[:2], counts=[1, 1])
    got = cache.read(first=[30, 7], fields=("positions",))["positions"]
    assert got.cpu().tolist() == [[30, 30], [7, 7]]


def test_read_of_ranges_and_types():
    torch = _torch()
    _case("read: ranges that start and end inside tiles, 16-bit results")
    pair = Pair(2, 2, 96, 64, "fp8")
    k, v = _rand((300, 2, 96), "float32", 6), _rand((300, 2, 96), "float32", 7)
    pair.append(k, v, [0, 1], [201, 99])
    for first, counts in ([3, 0], [1, 99]), ([31, 33], [34, 0]), ([64, 98], [137, 1]), ([201, 99], [0, 0]):
        got = pair.cache.read(first=first, counts=counts, fields=("v", "k"), dtype=torch.bfloat16)
        for name, stores in (("k", pair.k), ("v", pair.v)):
            want = np.concatenate([stores[s].values32()[f:f + n]
                                   for s, (f, n) in enumerate(zip(first, counts))])
            assert torch.equal(got[name].cpu(), torch.from_numpy(want).to(torch.bfloat16))


def test_truncate_returns_blocks_and_keeps_scales():
    _case("truncate, append again, empty")
    pair = Pair(2, 2, 64, 32, "int8", blocks=8)
    big = _rand((100, 2, 64), "float32", 8, 10.0)
    small = _rand((60, 2, 64), "float32", 9, 0.1)
    pair.append(big, big, [0], [100])
    assert pair.cache.info()["free_blocks"] == 4
    pair.cache.truncate([40, 0])
    assert pair.cache.info()["free_blocks"] == 6
    for st in (pair.k[0], pair.v[0]):
        st.codes, st.scales = st.codes[:40], st.scales[:2]
    pair.append(small, small, [0], [60])  # the begun block keeps the scale of the large ones
    pair.check_values()
    pair.cache.truncate(0)
    assert pair.cache.info()["free_blocks"] == 8 and not pair.cache.lengths.any()
    for st in (pair.k[0], pair.v[0]):
        st.codes, st.scales = st.codes[:0], st.scales[:0]
    pair.append(small, small, [0], [60])
    pair.check_values()


# ---- attention ------------------------------------------------------------------


@pytest.mark.parametrize("code", ["int8", "fp8"])
@pytest.mark.parametrize("dtype", ["bfloat16", "float16", "float32"])
@pytest.mark.parametrize("heads,group,dim,block", [(2, 1, 64, 32), (1, 7, 40, 32), (2, 4, 128, 64),
                                                   (1, 3, 96, 128), (1, 16, 192, 64),
                                                   (1, 20, 256, 256)])
def test_step_attention(code, dtype, heads, group, dim, block):
    """One token of sequences of 1, 31, 32, 33, 0 and 700 slots."""
    lens = [1, 31, 32, 33, 0, 700]
    _case(f"step {code} {dtype} heads {heads} x {group} dim {dim} block {block} lens {lens}")
    pair = Pair(6, heads, dim, block, code, blocks=40)
    pair.append(_rand((sum(lens), heads, dim), dtype, 20, 0.7), _rand((sum(lens), heads, dim), dtype, 21),
                list(range(6)), lens)
    q = _rand((6, heads * group, dim), dtype, 22)
    _check_attend(pair, q, list(range(6)), [1] * 6)
    # another order, not all of them
    _check_attend(pair, q[:3], [5, 0, 3], [1] * 3, decay=1.0)
    _check_attend(pair, q[:2], [5, 3], [1] * 2, decay=0.5, scale=0.3)


@pytest.mark.parametrize("code", ["int8", "fp8"])
@pytest.mark.parametrize("dtype", ["bfloat16", "float16", "float32"])
@pytest.mark.parametrize("dim", [64, 80, 128, 192, 256])
@pytest.mark.parametrize("group,counts", [(1, [5, 0, 17]), (4, [40, 3, 130])])
def test_chunk_attention(code, dtype, dim, group, counts):
    lens = [77, 3, 150]
    _case(f"chunk {code} {dtype} dim {dim} group {group} counts {counts} of {lens}")
    pair = Pair(3, 2, dim, 32, code)
    pair.append(_rand((230, 2, dim), dtype, 30, 0.7), _rand((230, 2, dim), dtype, 31), [0, 1, 2], lens)
    q = _rand((sum(counts), 2 * group, dim), dtype, 32)
    _check_attend(pair, q, [0, 1, 2], counts)
    _check_attend(pair, q, [0, 1, 2], counts, window=33, decay=1.0)
    _check_attend(pair, q, [0, 1, 2], counts, causal=False, decay=0.0)


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
@pytest.mark.parametrize("window", [1, 31, 32, 65, 1000])
@pytest.mark.parametrize("counts", [[1, 1], [6, 2], [90, 33]])
@pytest.mark.parametrize("causal", [True, False])
def test_windows(dtype, window, counts, causal):
    _case(f"window {window} counts {counts} causal {causal} {dtype}")
    pair = Pair(2, 1, 64, 32, "int8")
    pair.append(_rand((420, 1, 64), dtype, 40, 0.7), _rand((420, 1, 64), dtype, 41), [0, 1], [333, 87])
    _check_attend(pair, _rand((sum(counts), 3, 64), dtype, 42), [0, 1], counts, window=window,
                  causal=causal, decay=0.0)


@pytest.mark.parametrize("counts", [[1, 1], [9, 4], [70, 20]])
@pytest.mark.parametrize("form", ["bool", "uint8", "transposed", "broadcast"])
def test_masks_and_rows_that_see_nothing(counts, form):
    torch = _torch()
    _case(f"mask {form} counts {counts}")
    pair = Pair(2, 2, 64, 32, "fp8")
    pair.append(_rand((190, 2, 64), "bfloat16", 50, 0.7), _rand((190, 2, 64), "bfloat16", 51), [0, 1], [130, 60])
    t = sum(counts)
    g = torch.Generator().manual_seed(52)
    mask = (torch.rand((t, 131), generator=g) < 0.3).to("cuda:0")
    mask[0] = False      # a row without a slot
    mask[t - 1, :40] = False
    if form == "uint8":
        mask = mask.to(torch.uint8) * 7
    elif form == "transposed":
        mask = mask.t().contiguous().t()
    elif form == "broadcast":
        mask = mask[1:2].expand(t, 131)
    q = _rand((t, 4, 64), "bfloat16", 53)
    _check_attend(pair, q, [0, 1], counts, mask=mask, decay=1.0)
    _check_attend(pair, q, [0, 1], counts, mask=mask, causal=False, window=50)


def test_more_tokens_than_slots_leaves_rows_empty():
    _case("counts above the length")
    pair = Pair(2, 1, 64, 32, "int8")
    pair.append(_rand((5, 1, 64), "float32", 60), _rand((5, 1, 64), "float32", 61), [0], [5])
    _check_attend(pair, _rand((12, 2, 64), "float32", 62), [0, 1], [9, 3], decay=1.0)


@pytest.mark.parametrize("n,group,dtype", [(20_011, 8, "bfloat16"), (9_000, 1, "float32")])
def test_long_sequence_goes_over_many_workgroups(n, group, dtype):
    _case(f"long: {n} slots, group {group} {dtype}")
    pair = Pair(1, 2, 64, 64, "int8", blocks=320)
    pair.append(_rand((n, 2, 64), dtype, 70, 0.7), _rand((n, 2, 64), dtype, 71), [0], [n])
    _check_attend(pair, _rand((1, 2 * group, 64), dtype, 72), [0], [1], decay=1.0)
    _check_attend(pair, _rand((40, 2 * group, 64), dtype, 73), [0], [40], decay=1.0)


def test_scores_far_apart_and_value_scales_far_apart():
    """Largest scores at the end, in the middle and at the start; blocks whose values
    differ by 2^40; a block of zeros."""
    _case("running reference")
    for where in (0, 100, 318):
        pair = Pair(1, 1, 64, 32, "int8")
        k = _rand((320, 1, 64), "float32", 80, 0.3)
        v = _rand((320, 1, 64), "float32", 81)
        v[64:96] *= 2.0 ** 20
        v[128:160] *= 2.0 ** -20
        v[160:192] = 0
        k[192:224] = 0
        q = _rand((3, 1, 64), "float32", 82)
        k[where] = q[0] * 6.0
        pair.append(k, v, [0], [320])
        _check_attend(pair, q, [0], [3], decay=0.0)


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
@pytest.mark.parametrize("size", [-30, -20, 0, 20])
@pytest.mark.parametrize("n,counts", [(320, 3), (320, 150), (1 << 13, 600)])
def test_blocks_of_zeros_beside_values_of_any_size(dtype, size, n, counts):
    """The zeros, first and in the middle, are the slots that the rows see best."""
    _case(f"zeros beside 2^{size} {dtype} {n} {counts}")
    pair = Pair(1, 1, 64, 32, "int8", blocks=n // 32)
    k = _rand((n, 1, 64), "float32", 83, 0.3)
    v = _rand((n, 1, 64), "float32", 84) * 2.0 ** size
    q = _rand((counts, 8, 64), dtype, 89)
    for at in (0, 160):
        v[at:at + 32] = 0
        k[at:at + 32] *= 4
    pair.append(k, v, [0], [n])
    _check_attend(pair, q, [0], [counts], decay=0.0)


@pytest.mark.parametrize("code", ["int8", "fp8"])
@pytest.mark.parametrize("size,n,counts", [(-102, 100_000, 2), (-101, 9000, 300), (120, 3000, 2), (120, 3000, 300)])
def test_smallest_and_largest_value_scales(code, size, n, counts):
    _case(f"values of 2^{size} {code} {n} {counts}")
    pair = Pair(1, 1, 64, 64, code, blocks=n // 64 + 1)
    k = _rand((n, 1, 64), "float32", 90, 0.02)
    v = _rand((n, 1, 64), "float32", 91) * 2.0 ** size
    pair.append(k, v, [0], [n])
    _check_attend(pair, _rand((counts, 2, 64), "float32", 92), [0], [counts], decay=0.0)


@pytest.mark.parametrize("code", ["int8", "fp8"])
@pytest.mark.parametrize("dtype", ["bfloat16", "float16", "float32"])
@pytest.mark.parametrize("group", [1, 40, 130])
def test_logarithms_and_weights_keep_float32_whatever_the_query_type(code, dtype, group):
    """One dimension and few slots: the bounds come down to some 2^-14, below what a half
    precision probability in the denominator would cost."""
    lens = [2, 3, 5, 9, 17]
    _case(f"logarithms {code} {dtype} group {group}")
    pair = Pair(5, 1, 1, 32, code)
    pair.append(_rand((sum(lens), 1, 1), dtype, 86), _rand((sum(lens), 1, 1), dtype, 87), list(range(5)), lens)
    q = _rand((5, group, 1), dtype, 88)
    _check_attend(pair, q, list(range(5)), [1] * 5, decay=0.0, scale=0.5)
    _check_attend(pair, q, list(range(5)), [1] * 5, scale=0.5)


@pytest.mark.parametrize("n,group,counts", [(3000, 4, [120, 30]), (2100, 8, [70, 1]), (5000, 1, [300, 260])])
@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
def test_many_rows_over_long_sequences(n, group, counts, dtype):
    """Enough rows and tiles for the kernel of many rows, in one or several splits."""
    _case(f"many rows: {n} slots group {group} counts {counts} {dtype}")
    pair = Pair(2, 2, 64, 64, "fp8", blocks=200)
    pair.append(_rand((n + 900, 2, 64), dtype, 74, 0.7), _rand((n + 900, 2, 64), dtype, 75), [0, 1], [n, 900])
    q = _rand((sum(counts), 2 * group, 64), dtype, 76)
    _check_attend(pair, q, [0, 1], counts)
    _check_attend(pair, q, [0, 1], counts, window=1000, decay=1.0)
    mask = (_torch().rand((sum(counts), n), generator=_torch().Generator().manual_seed(77)) < 0.5).to("cuda:0")
    _check_attend(pair, q, [0, 1], counts, mask=mask)


def test_rows_of_any_size():
    """Queries from 2^-60 to 2^60, and zero: the scale undoes it."""
    torch = _torch()
    _case("query magnitudes")
    pair = Pair(1, 1, 64, 32, "fp8")
    pair.append(_rand((100, 1, 64), "float32", 83), _rand((100, 1, 64), "float32", 84), [0], [100])
    for e in (-60, 60):
        _check_attend(pair, _rand((2, 4, 64), "float32", 85) * 2.0 ** e, [0], [2], scale=0.125 * 2.0 ** -e)
    _check_attend(pair, torch.zeros((2, 4, 64), device="cuda:0"), [0], [2], decay=1.0)


def test_non_finite_tokens_stay_in_their_block_and_head():
    torch = _torch()
    _case("NaN and infinities in the cache and in queries")
    for bad in (float("nan"), float("inf"), float("-inf")):
        for code in ("int8", "fp8"):
            pair = Pair(1, 2, 64, 32, code)
            k, v = _rand((100, 2, 64), "bfloat16", 90), _rand((100, 2, 64), "bfloat16", 91)
            k[40, 0, 5] = bad
            v[70, 1, 63] = bad
            pair.append(k[:90], v[:90], [0], [90])
            pair.append(k[90:], v[90:], [0], [10])
            pair.check_values()
            q = _rand((1, 4, 64), "bfloat16", 92)
            out = pair.cache.attend(q, decay=1.0)
            assert torch.isnan(out).all()
            # a window behind the blocks, and a mask over them
            _check_attend(pair, q, [0], [1], window=4)
            mask = torch.ones((1, 100), dtype=torch.bool, device="cuda:0")
            mask[:, 32:96] = False
            _check_attend(pair, q, [0], [1], mask=mask)
            mask[:, 64:96] = True  # head 0 sees nothing bad, head 1 does
            out = pair.cache.attend(q, mask=mask)
            assert torch.isfinite(out[:, :2]).all() and torch.isnan(out[:, 2:]).all()
            many = q.expand(70, 4, 64)
            out = pair.cache.attend(many, window=4, causal=False)
            assert torch.isnan(out[0]).all() and torch.isfinite(out[-1]).all()
            pair.cache.truncate(0)
            for st in (pair.k[0], pair.v[0]):
                st.codes, st.scales = st.codes[:0], st.scales[:0]
            k[40, 0, 5] = v[70, 1, 63] = 0
            pair.append(k, v, [0], [100])  # the blocks are used again
            _check_attend(pair, q, [0], [1])
            q2 = q.clone()
            q2[0, 1, 3] = bad
            out = pair.cache.attend(q2)
            assert torch.isnan(out[0, 1]).all()
            assert torch.isfinite(out[0, [0, 2, 3]]).all()


def test_nan_seen_by_one_part_of_a_long_row_reaches_its_result():
    torch = _torch()
    _case("NaN in one split of a long sequence")
    pair = Pair(1, 1, 64, 32, "int8", blocks=400)
    k, v = _rand((12_000, 1, 64), "bfloat16", 93), _rand((12_000, 1, 64), "bfloat16", 94)
    k[7000, 0, 0] = float("nan")
    pair.cache.append(k, v)
    for t in (1, 80):
        out, lse = pair.cache.attend(_rand((t, 1, 64), "bfloat16", 95), return_lse=True)
        assert torch.isnan(out).all() and torch.isnan(lse).all()


# ---- eviction ---------------------------------------------------------------------


def _check_evict(pair, weights, seqs, lens, budget, recent, into=None, dropped=True):
    torch = _torch()
    before = [(pair.k[s], pair.v[s]) for s in seqs]
    gone = pair.cache.evict(budget, recent, seqs=seqs, into=into, dropped=dropped)
    most = max(max(lens) - budget, 0)
    at = 0
    for i, (s, n) in enumerate(zip(seqs, lens)):
        w = weights[at:at + n]
        at += n
        stay, left = ref.keep_slots(w, budget, recent)
        heads = np.arange(pair.heads)[None]
        to = s if into is None else into[i]
        cut = n > budget
        for name, stores, old in (("k", pair.k, before[i][0]), ("v", pair.v, before[i][1])):
            stores[to] = old.kept(stay) if cut or into is not None else old
            if dropped:
                want = np.zeros((most, pair.heads, pair.dim), np.float32)
                want[:len(left)] = old.values32()[left, heads]
                assert np.array_equal(_np(gone[name][i]), want, equal_nan=True), (name, s)
        if dropped:
            want = np.full((most, pair.heads), -1)
            want[:len(left)] = left
            assert np.array_equal(gone["positions"][i].cpu().numpy(), want)
        got = pair.cache.read(seqs=[to])
        assert np.array_equal(got["positions"].cpu().numpy(), stay)
        assert np.array_equal(_np(got["weights"]), w[stay, heads], equal_nan=True)
    pair.check_values(seqs if into is None else list(seqs) + list(into))


@pytest.mark.parametrize("code", ["int8", "fp8"])
@pytest.mark.parametrize("heads,dim,block", [(2, 64, 32), (3, 40, 64), (1, 256, 128), (2, 128, 256)])
@pytest.mark.parametrize("budget,recent", [(1, 0), (64, 0), (100, 30), (100, 100), (97, 1), (0, 0)])
@pytest.mark.parametrize("in_place", [True, False])
def test_evict(code, heads, dim, block, budget, recent, in_place):
    torch = _torch()
    lens = [333, 20, 101, 0]
    _case(f"evict {code} heads {heads} dim {dim} block {block} budget {budget} recent {recent} "
          f"in place {in_place}")
    pair = Pair(8, heads, dim, block, code, blocks=64)
    t = sum(lens)
    g = torch.Generator().manual_seed(100)
    w = torch.rand((t, heads), generator=g)
    w = torch.where(w < 0.5, (w * 8).round() / 8, w)  # many equal ones
    w[::17] = 0.0
    k = _rand((t, heads, dim), "float32", 101) * (1 + torch.arange(t, device="cuda:0")[:, None, None] % 5)
    pair.append(k, k.flip(0), [0, 1, 2, 3], lens, weights=w.to("cuda:0"))
    _check_evict(pair, w.numpy(), [0, 1, 2, 3], lens, budget, recent,
                 into=None if in_place else [4, 5, 6, 7])
    if in_place and budget:
        # the cut sequences go on
        more = _rand((40, heads, dim), "float32", 102)
        pair.append(more, more, [0, 1], [33, 7])
        pair.check_values()
        got = pair.cache.read(seqs=[0], fields=("positions",))["positions"]
        assert got[-1].cpu().tolist() == [365] * heads
        _check_attend(pair, _rand((2, heads, dim), "float32", 103), [0, 1], [1, 1], decay=1.0)


def test_evict_orders_odd_weights():
    """NaN above infinity above numbers, -0 equal to 0, negative ones last."""
    torch = _torch()
    _case("evict: NaN, infinities, signed zeros, negative weights")
    w = np.array([0.0, -0.0, np.nan, 3.0, np.inf, -2.0, -np.inf, 0.0, np.nan, 1e-40], np.float32)[:, None]
    for budget in range(11):
        pair = Pair(1, 1, 32, 32, "int8")
        k = _rand((10, 1, 32), "float32", 104)
        pair.append(k, k, [0], [10], weights=torch.from_numpy(w).to("cuda:0"))
        _check_evict(pair, w, [0], [10], budget, 0)


def test_evict_long_sequence_and_in_place_without_spare_blocks():
    torch = _torch()
    _case("evict 40000 slots; sequences cut one after the other in a full pool")
    pair = Pair(1, 2, 64, 64, "int8", blocks=720)
    g = torch.Generator().manual_seed(105)
    w = (torch.rand((40_000, 2), generator=g) * 1000).floor()  # about 40 of each
    k = _rand((40_000, 2, 64), "bfloat16", 106)
    pair.append(k, k, [0], [40_000], weights=w.to("cuda:0"))
    _check_evict(pair, w.numpy(), [0], [40_000], 5_001, 77)
    # 4 sequences of 3 blocks in a pool of 13: one free block at a time
    pair = Pair(4, 1, 64, 32, "fp8", blocks=13)
    w = torch.rand((4 * 96, 1), generator=g)
    k = _rand((4 * 96, 1, 64), "float32", 107)
    pair.append(k, k, [0, 1, 2, 3], [96] * 4, weights=w.to("cuda:0"))
    _check_evict(pair, w.numpy(), [0, 1, 2, 3], [96] * 4, 32, 8)
    assert pair.cache.info()["free_blocks"] == 9


def test_evict_to_a_budget_far_above_the_lengths():
    """What the call holds follows the sequences, not the budget: 17 of 2^30 would take 1.1 TB."""
    torch = _torch()
    _case("evict with a budget of 2^30")
    pair = Pair(34, 8, 64, 32, "int8", blocks=64)
    lens = [2 + i for i in range(17)]
    k = _rand((sum(lens), 8, 64), "bfloat16", 112)
    pair.append(k, k.flip(0), list(range(17)), lens)
    want = pair.cache.read(seqs=list(range(17)))
    budget = 2 ** 30 - 1
    pair.cache.evict(budget, recent=budget, seqs=list(range(17)), into=list(range(17, 34)))
    got = pair.cache.read(seqs=list(range(17, 34)))
    for name in ("k", "v", "positions", "weights"):
        assert torch.equal(got[name], want[name]), name


def test_evict_keeps_poisoned_slots_poisoned():
    torch = _torch()
    _case("evict with NaN scales")
    pair = Pair(1, 1, 64, 32, "int8")
    k = _rand((128, 1, 64), "float32", 108)
    k[5] = float("nan")
    w = torch.zeros((128, 1))
    w[[1, 40, 41, 100]] = 1.0
    pair.append(k, k, [0], [128], weights=w.to("cuda:0"))
    _check_evict(pair, w.numpy(), [0], [128], 4, 0)
    assert torch.isnan(pair.cache.read()["k"]).all()


# ---- large offsets, streams, many sequences ------------------------------------------


def test_offsets_beyond_32_bits():
    """A pool of 5 GiB, the used slots at its end."""
    torch = _torch()
    _case("5 GiB pool")
    import vicinity_amd as va

    heads, dim = 16, 256  # 8 KiB a slot
    n = 5 * 2 ** 30 // (2 * heads * dim)
    cache = va.KVCache(2, heads, dim, n // 256 + 2, block_tokens=256)
    row = _rand((1, heads, dim), "bfloat16", 110)
    cache.append(row.expand(n, heads, dim), row.expand(n, heads, dim), seqs=[0])
    pair = Pair(1, heads, dim, 256, "int8")
    k, v = _rand((300, heads, dim), "bfloat16", 111), _rand((300, heads, dim), "bfloat16", 112)
    pair.append(k, v, [0], [300])
    cache.append(k, v, seqs=[1])
    q = _rand((1, heads, dim), "bfloat16", 113)
    assert torch.equal(cache.attend(q, seqs=[1]), pair.cache.attend(q))
    want = pair.check_values()
    got = cache.read(seqs=[1])
    assert all(torch.equal(got[f], want[f]) for f in got)
    # every slot of the long one holds the same value
    out = cache.attend(q, seqs=[0]).float()
    one = cache.read(seqs=[0], first=[n - 1], counts=[1])
    assert (out - one["v"][0]).abs().max() <= 2.0 ** -8 * one["v"].abs().max()
    tail = cache.read(seqs=[0], first=[n - 700], counts=[700])
    assert (tail["k"] == one["k"]).all() and (tail["v"] == one["v"]).all()


def test_more_sequences_than_one_launch_takes():
    torch = _torch()
    _case("300 sequences")
    n = 300
    pair = Pair(n, 1, 64, 32, "int8", blocks=700)
    lens = [(7 * i) % 70 for i in range(n)]
    t = sum(lens)
    order = [(i * 7) % n for i in range(n)]
    pair.append(_rand((t, 1, 64), "float16", 120), _rand((t, 1, 64), "float16", 121), order, lens)
    pair.check_values(order)
    _check_attend(pair, _rand((n, 2, 64), "float16", 122), order, [1] * n, decay=1.0)
    pair.cache.evict(20, 5)
    assert list(pair.cache.lengths) == [min(len(pair.k[i].codes), 20) for i in range(n)]


def test_calls_on_different_streams_follow_one_another():
    torch = _torch()
    _case("streams")
    import vicinity_amd as va

    k, v = _rand((3000, 2, 64), "bfloat16", 130), _rand((3000, 2, 64), "bfloat16", 131)
    q = _rand((1, 4, 64), "bfloat16", 132)
    want_cache = va.KVCache(1, 2, 64, 100)
    for i in range(0, 3000, 100):
        want_cache.append(k[i:i + 100], v[i:i + 100])
    want = want_cache.attend(q)
    cache = va.KVCache(1, 2, 64, 100)
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    for i in range(0, 3000, 100):
        cache.append(k[i:i + 100], v[i:i + 100], stream=a if i % 200 else b)
    out = cache.attend(q, stream=a)
    a.synchronize()
    assert torch.equal(out, want)
    with torch.cuda.stream(b):
        again = cache.attend(q)
    b.synchronize()
    assert torch.equal(again, want)


def test_repeated_calls_give_the_same_bits():
    torch = _torch()
    _case("determinism")
    pair = Pair(1, 2, 128, 64, "int8", blocks=160)
    pair.append(_rand((9000, 2, 128), "bfloat16", 140), _rand((9000, 2, 128), "bfloat16", 141), [0], [9000])
    for t in (1, 33):
        q = _rand((t, 8, 128), "bfloat16", 142)
        first, w = pair.cache.attend(q, decay=0.0), pair.cache.read(fields=("weights",))["weights"]
        for _ in range(3):
            assert torch.equal(pair.cache.attend(q, decay=0.0), first)
            assert torch.equal(pair.cache.read(fields=("weights",))["weights"], w)


@pytest.mark.parametrize("rows", [0, 1, 70])
def test_sequences_without_query_tokens_only_decay(rows):
    """No token at all, one of an empty sequence, 70 of the first (a second pass over the keys,
    and a second launch without rows)."""
    torch = _torch()
    _case(f"weights without tokens, {rows} rows")
    import vicinity_amd as va

    n, lens = 130, [0] + [40 + i for i in range(129)]
    if rows > 1:
        lens[0] = 100
    cache = va.KVCache(n, 2, 64, 6 * n, block_tokens=32)
    x = _rand((sum(lens), 2, 64), "bfloat16", 180)
    w = torch.rand((sum(lens), 2), device="cuda:0")
    cache.append(x, x, counts=lens, weights=w)
    q = _rand((rows, 2, 64), "bfloat16", 181)
    out = cache.attend(q, counts=[rows] + [0] * (n - 1), decay=0.5)
    assert out.shape == q.shape and torch.isfinite(out).all()
    got = cache.read(fields=("weights",))["weights"]
    assert torch.equal(got[lens[0]:], 0.5 * w[lens[0]:])
    gave = (got - 0.5 * w)[:lens[0]].sum(0)
    assert torch.allclose(gave, torch.full_like(gave, float(rows if lens[0] else 0)), rtol=1e-4)


# ---- refusals --------------------------------------------------------------------------


def test_refusals_leave_the_cache_as_it_was():
    torch = _torch()
    _case("refusals")
    import vicinity_amd as va
    from vicinity_amd import _lib

    cache = va.KVCache(3, 2, 64, 6, block_tokens=32, max_blocks=4)
    x = _rand((40, 2, 64), "bfloat16", 150)
    cache.append(x, x, seqs=[0])
    q = _rand((1, 4, 64), "bfloat16", 151)

    def refused(kind, match, f, *args, **kw):
        with pytest.raises(kind, match=match) as e:
            f(*args, **kw)
        return e.value

    big = _rand((1, 2, 64), "bfloat16", 152).expand(200, 2, 64)
    refused(ValueError, "max_blocks", cache.append, big, big, seqs=[0])
    err = refused(_lib.VicinityGpuError, "more blocks", cache.append, big[:192], big[:192], seqs=[1, 2])
    assert err.code == _lib.ERR_OUT_OF_MEMORY
    refused(ValueError, "out of range", cache.append, x, x, seqs=[3])
    refused(ValueError, "twice", cache.append, x, x, seqs=[0, 0])
    refused(ValueError, "counts", cache.append, x, x, seqs=[0, 1], counts=[3, 4])
    refused(ValueError, "counts", cache.append, x, x, seqs=[0, 1], counts=[-1, 41])
    refused(ValueError, "counts", cache.append, x[:1], x[:1], seqs=[0, 1])
    refused(ValueError, "shape", cache.append, x[:, :1], x[:, :1], seqs=[0])
    refused(ValueError, "same shape", cache.append, x, x.float(), seqs=[0])
    refused(TypeError, "float32, float16 or bfloat16", cache.append, x.double(), x.double(), seqs=[0])
    refused(TypeError, "tensor", cache.append, x.float().cpu().numpy(), x, seqs=[0])
    refused(ValueError, "GPU", cache.append, x.cpu(), x.cpu(), seqs=[0])
    refused(TypeError, "int32", cache.append, x, x, seqs=[0], positions=torch.zeros((40, 2), device="cuda:0"))
    refused(ValueError, "contiguous", cache.append, x, x, seqs=[0],
            weights=torch.zeros((2, 40), device="cuda:0").t())
    refused(ValueError, "multiple", cache.attend, q[:, :3], seqs=[0])
    refused(ValueError, "shape", cache.attend, q[:, :, :32], seqs=[0])
    refused(ValueError, "window", cache.attend, q, seqs=[0], window=-1)
    refused(ValueError, "scale", cache.attend, q, seqs=[0], scale=float("nan"))
    refused(ValueError, "decay", cache.attend, q, seqs=[0], decay=float("inf"))
    refused(ValueError, "mask", cache.attend, q, seqs=[0], mask=torch.ones((1, 40), device="cuda:0"))
    refused(ValueError, "longest", cache.attend, q, seqs=[0],
            mask=torch.ones((1, 39), device="cuda:0", dtype=torch.bool))
    refused(ValueError, "out must", cache.attend, q, seqs=[0], out=torch.empty_like(q).float())
    refused(ValueError, "recent", cache.evict, 4, 5)
    refused(ValueError, "budget", cache.evict, -1)
    refused(ValueError, "not empty", cache.evict, 4, 0, seqs=[1], into=[0])
    refused(ValueError, "twice", cache.evict, 4, 0, seqs=[0], into=[0])
    refused(ValueError, "into names", cache.evict, 4, 0, seqs=[0], into=[1, 2])
    refused(ValueError, "outside", cache.read, seqs=[0], first=[10], counts=[31])
    refused(ValueError, "fields", cache.read, fields=("q",))
    refused(TypeError, "dtype", cache.read, dtype=torch.int8)
    refused(ValueError, "outside", cache.truncate, [41], seqs=[0])
    refused(ValueError, "one entry", cache.truncate, [1, 2], seqs=[0])
    for kw in (dict(head_dim=257), dict(block_tokens=48), dict(code="int4"), dict(num_seqs=0),
               dict(num_blocks=0), dict(num_heads=0)):
        args = dict(num_seqs=1, num_heads=1, head_dim=64, num_blocks=1) | kw
        refused(ValueError, "must be", va.KVCache, **args)
    # in a full pool a cut finds no block
    cache.append(big[:128], big[:128], seqs=[1])
    err = refused(_lib.VicinityGpuError, "free blocks", cache.evict, 32, 0, seqs=[1])
    assert err.code == _lib.ERR_OUT_OF_MEMORY
    assert list(cache.lengths) == [40, 128, 0]
    got = cache.read(seqs=[0])
    one = va.KVCache(1, 2, 64, 6, block_tokens=32)
    one.append(x, x)
    assert all(torch.equal(a, b) for a, b in zip(got.values(), one.read().values()))


def test_calls_of_more_workgroups_than_a_launch_can_have():
    """4096 heads: 40960 tokens enter 10.5 M parts of the pool, two such sequences take two launches."""
    torch = _torch()
    _case("4096 heads, 2 x 40960 tokens")
    import vicinity_amd as va

    heads, n = 4096, 40960
    cache = va.KVCache(2, heads, 1, 2 * n // 32 + 2, block_tokens=32, max_blocks=2560)
    k = (torch.arange(2 * n, device="cuda:0") % 128).to(torch.float16)[:, None, None]
    k = torch.where(k == 0, 127, k)  # and every block's scale is 1
    k[::32] = 127
    k = k.expand(2 * n, heads, 1)
    with pytest.raises(ValueError, match="one sequence in one call"):
        cache.append(k[:65600], k[:65600], seqs=[0])
    assert cache.lengths.tolist() == [0, 0]
    cache.append(k, k, seqs=[0, 1], counts=[n, n])
    for field in ("k", "v"):
        got = cache.read(seqs=[0, 1], fields=(field,), dtype=torch.float16)[field]
        assert torch.equal(got, k), field


def test_capture_is_refused():
    torch = _torch()
    _case("stream capture")
    import vicinity_amd as va
    from vicinity_amd import _lib

    cache = va.KVCache(1, 2, 64, 6)
    x = _rand((40, 2, 64), "bfloat16", 160)
    cache.append(x, x)
    q = _rand((1, 4, 64), "bfloat16", 161)
    want = cache.attend(q)
    torch.cuda.synchronize()
    out = torch.empty_like(q)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        with pytest.raises(ValueError, match="captured") as e:
            cache.attend(q, out=out)
        out.zero_()
    assert e.value.code == _lib.ERR_UNSUPPORTED
    assert torch.equal(cache.attend(q), want)


def test_allocation_failure_reports_and_recovers():
    torch = _torch()
    _case("device allocation failure")
    import vicinity_amd as va
    from vicinity_amd import _lib

    lib = _lib.load()
    for after in range(6):
        _lib.check(lib.vgpu_test_fail_device_allocations(after, 1))
        try:
            with pytest.raises(_lib.VicinityGpuError) as e:
                va.KVCache(1, 2, 64, 200)
            assert e.value.code == _lib.ERR_OUT_OF_MEMORY
        finally:
            _lib.check(lib.vgpu_test_fail_device_allocations(0, 0))
    cache = va.KVCache(1, 2, 64, 200)
    x = _rand((9000, 2, 64), "bfloat16", 170)
    cache.append(x, x)
    q = _rand((1, 2, 64), "bfloat16", 171)
    _lib.check(lib.vgpu_test_fail_device_allocations(0, 1))
    try:
        with pytest.raises(_lib.VicinityGpuError):
            cache.attend(q, decay=1.0)
    finally:
        _lib.check(lib.vgpu_test_fail_device_allocations(0, 0))
    assert not cache.read(fields=("weights",))["weights"].any()
    assert torch.isfinite(cache.attend(q, decay=1.0)).all()


def test_a_later_launch_without_memory_leaves_the_weights():
    """130 sequences take two launches; only the second needs more workspace than there is."""
    torch = _torch()
    _case("allocation failure, second launch")
    import vicinity_amd as va
    from vicinity_amd import _lib

    cache = va.KVCache(130, 2, 64, 129 + 300)
    x = _rand((130, 2, 64), "bfloat16", 172)
    cache.append(x, x)
    q = _rand((130, 2, 64), "bfloat16", 173)
    cache.attend(q, decay=1.0)
    more = _rand((9000, 2, 64), "bfloat16", 174)
    cache.append(more, more, seqs=[129])
    before = cache.read(fields=("weights",))["weights"]
    lib = _lib.load()
    _lib.check(lib.vgpu_test_fail_device_allocations(0, 1))
    try:
        with pytest.raises(_lib.VicinityGpuError) as e:
            cache.attend(q, decay=1.0)
        assert e.value.code == _lib.ERR_OUT_OF_MEMORY
    finally:
        _lib.check(lib.vgpu_test_fail_device_allocations(0, 0))
    assert torch.equal(cache.read(fields=("weights",))["weights"], before)
    cache.attend(q, decay=1.0)
    # every row gives its head a weight of 1 in all
    gave = (cache.read(fields=("weights",))["weights"] - before).sum(0)
    assert torch.allclose(gave, torch.full_like(gave, 130.0), rtol=1e-4)
