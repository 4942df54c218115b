"""Attention over values of any magnitude: blocks of zeros beside very small and very large
values, the smallest scales under scores that rise after the first tile, and value scales that
rise, fall or alternate along a sequence.  The bounds are those of the attention's own tests:
e = (D + 16) u (A + 32) in every probability, p's rounding, n (2 u + 2^-30) for the sums."""

import math

import numpy as np
import pytest

from test_gpu_kv import OUT_EPS, U, Pair, _case, _check_attend, _rand, _torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
@pytest.mark.parametrize("size", [-95, -60, 90, 110])
@pytest.mark.parametrize("n,counts", [(320, 3), (320, 150), (1 << 13, 600)])
def test_blocks_of_zeros_beside_the_smallest_and_the_largest_values(dtype, size, n, counts):
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


def _check_one_head(cache, q, out, lse, scale):
    """Row 0 of head 0 against float64 over the values that the cache holds; every row of
    every head got the same query and the same tokens."""
    torch = _torch()
    assert torch.equal(out, out[:1, :1].expand_as(out))
    assert torch.equal(lse, lse[:1, :1].expand_as(lse))
    held = cache.read(fields=("k", "v"))
    k, v = held["k"][:, 0].double().cpu().numpy(), held["v"][:, 0].double().cpu().numpy()
    q = q[0, 0].double().cpu().numpy()
    s = k @ q * scale
    m = s.max()
    p = np.exp(s - m)
    want, wlse = p @ v / p.sum(), m + math.log(p.sum())
    n, dim = k.shape
    e = (dim + 16) * U * (scale * (np.abs(k) @ np.abs(q)).max() + 32)
    name = str(out.dtype).split(".")[1]
    rel = 2 * e + (2.0 ** -22 if name == "float32" else 2.0 ** -11) + n * (2 * U + 2.0 ** -30)
    vmax = np.abs(v).max()
    err = np.abs(out[0, 0].double().cpu().numpy() - want)
    assert (err <= vmax * rel + OUT_EPS[name] * (np.abs(want) + vmax * rel)).all(), float(err.max() / vmax)
    assert abs(float(lse[0, 0]) - wlse) <= 2 * e + n * 2 * U + 4 * U * abs(wlse)


# heads, query heads on each, slots: enough rows that a workgroup goes over all tiles (few
# rows) or half of them (many rows) in one part
FORMS = [(64, 192, 65536), (64, 1024, 32768)]


@pytest.mark.parametrize("code", ["int8", "fp8"])
@pytest.mark.parametrize("heads,group,n", FORMS)
def test_smallest_scales_under_scores_that_rise_after_the_first_tile(code, heads, group, n):
    """The later scores stand 7.9 (base 2) above the first tile's, just too little to move the
    running reference."""
    torch = _torch()
    _case(f"rising scores at 2^-100 {code} {heads} x {group} {n}")
    import vicinity_amd as va

    cache = va.KVCache(1, heads, 32, n // 32, block_tokens=32, code=code)
    k = torch.zeros((n, 1, 32), device="cuda:0")
    k[32:, :, 0] = 1.0
    v = torch.full((1, 1, 1), 2.0 ** -100, device="cuda:0")
    cache.append(k.expand(n, heads, 32), v.expand(n, heads, 32))
    q = torch.zeros((1, 1, 32), device="cuda:0", dtype=torch.bfloat16)
    q[..., 0] = 5.46875  # 7.8897 / log2(e)
    out, lse = cache.attend(q.expand(1, heads * group, 32), scale=1.0, return_lse=True)
    _check_one_head(cache, q, out, lse, 1.0)


@pytest.mark.parametrize("order", ["rising", "falling", "alternating", "zeros, rising"])
@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
@pytest.mark.parametrize("heads,group,n", FORMS)
def test_value_scales_far_apart_along_a_sequence(order, dtype, heads, group, n):
    """Blocks from 2^-100 to 2^110, in windows longer than the 64 tiles that a wave looks ahead."""
    torch = _torch()
    _case(f"scales {order} {dtype} {heads} x {group} {n}")
    import vicinity_amd as va

    cache = va.KVCache(1, heads, 32, n // 64, block_tokens=64, code="int8")
    k, v = _rand((n, 1, 32), "float32", 200, 0.3), _rand((n, 1, 32), "float32", 201)
    steps = torch.arange(n, device="cuda:0") // (n // 8)
    size = -100.0 + 30.0 * steps
    if order == "falling":
        size = size.flip(0)
    elif order == "alternating":
        size = torch.where(steps % 2 == 0, 110.0, -100.0)
    v *= torch.exp2(size)[:, None, None]
    if order == "zeros, rising":
        v[:n // 8] = 0
    cache.append(k.expand(n, heads, 32), v.expand(n, heads, 32))
    q = _rand((1, 1, 32), dtype, 202)
    out, lse = cache.attend(q.expand(1, heads * group, 32), return_lse=True)
    _check_one_head(cache, q, out, lse, float(np.float32(1 / math.sqrt(32))))


@pytest.mark.parametrize("counts", [3, 150])
def test_rows_that_lean_on_values_far_below_the_others(counts):
    """Values 2^-70 of the others with all of the weight: they are the result, to their own size."""
    torch = _torch()
    _case(f"small values seen best, {counts} tokens")
    pair = Pair(1, 1, 64, 32, "int8")
    k, v = _rand((320, 1, 64), "float32", 210, 0.05), _rand((320, 1, 64), "float32", 211)
    v[96:128] *= 2.0 ** -70
    pair.append(k, v, [0], [320])
    see = torch.zeros((counts, 320), dtype=torch.bool, device="cuda:0")
    see[:, 96:128] = True
    q = _rand((counts, 2, 64), "float32", 212)
    out = pair.cache.attend(q, mask=see, causal=False)
    small = Pair(1, 1, 64, 32, "int8")
    small.append(k[96:128], v[96:128], [0], [32])
    want = small.cache.attend(q, causal=False)
    size = small.cache.read(fields=("v",))["v"].abs().max()
    # 32 slots with scores of a few tenths, each in float32
    assert ((out - want).abs() <= 2.0 ** -17 * size).all()
