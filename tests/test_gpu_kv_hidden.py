"""Values that a row does not see, however large or small, have no part in its result: the
bounds of the attention's own tests, by the values that the row does see."""

import numpy as np
import pytest

import kv_reference as ref
from test_gpu_kv import OUT_EPS, U, Pair, _case, _np, _rand, _torch

pytestmark = pytest.mark.gpu


def _check(pair, q, see, **kw):
    """Each token by the largest value among the slots that it sees: see [t, n]."""
    dtype = str(q.dtype).split(".")[1]
    out, lse = pair.cache.attend(q, return_lse=True, **kw)
    k, v = pair.k[0].values(), pair.v[0].values()
    n, dim, t = len(k), pair.dim, len(q)
    scale = float(np.float32(1 / np.sqrt(dim)))
    want, wlse, w = ref.attend(_np(q).astype(np.float64), k, v, see, scale)
    g = q.shape[1] // pair.heads
    a = scale * (np.abs(_np(q)).max(0) * np.repeat(np.abs(k).max(0), g, axis=0)).sum(1).max()
    e = (dim + 16) * U * (a + 32)
    rel = 2 * e + (2.0 ** -22 if dtype == "float32" else 2.0 ** -11) + n * (2 * U + 2.0 ** -30)
    size = np.repeat(np.abs(v).max(2), g, axis=1)  # [n, heads]
    vmax = np.stack([size[row].max(0) if row.any() else np.zeros(size.shape[1]) for row in see])[:, :, None]
    err = np.abs(_np(out).astype(np.float64) - want)
    limit = vmax * rel + OUT_EPS[dtype] * (np.abs(want) + vmax * rel)
    assert (err <= limit).all(), (np.argwhere(err > limit)[:5].tolist(), float((err / np.maximum(vmax, 1e-300)).max()))
    seen = see.any(1)
    got = _np(lse).astype(np.float64)
    assert np.isneginf(got[~seen]).all()
    assert (np.abs(got - wlse)[seen] <= 2 * e + n * 2 * U + 4 * U * np.abs(wlse[seen])).all()
    if kw.get("decay") is not None:
        after = _np(pair.cache.read(fields=("weights",))["weights"])
        rows = t * g
        assert (np.abs(after - w) <= (3 * e + (n + rows + 8) * 2 * U) * w + rows * 2.0 ** -100).all()


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("big,size", [(120, 0), (60, -50), (120, -60), (-95, 0), (-95, 110)])
@pytest.mark.parametrize("n,counts", [(320, 2), (320, 150), (8192, 2), (8192, 300)])
def test_blocks_that_a_row_does_not_see(dtype, dim, big, size, n, counts):
    """A block of 2^big in the middle of values of 2^size, hidden from some of the rows by a mask, by
    the window or because it comes after them."""
    torch = _torch()
    _case(f"hidden 2^{big} beside 2^{size} {dtype} dim {dim} {n} {counts}")
    group = 4
    pair = Pair(1, 1, dim, 32, "int8", blocks=n // 32)
    k = _rand((n, 1, dim), "float32", 800, 0.2)
    v = _rand((n, 1, dim), "float32", 801)
    at = n - 96
    where = torch.zeros(n, device="cuda:0")
    where[:] = size
    where[at:at + 32] = big
    where[64:96] = -1000.0  # zeros
    v *= torch.exp2(where)[:, None, None]
    pair.append(k, v, [0], [n])
    q = _rand((counts, group, dim), dtype, 802)
    see = np.ones((counts, n), bool)
    see[::2, at:at + 32] = False
    mask = torch.from_numpy(see).to("cuda:0")
    _check(pair, q, see, mask=mask, causal=False, decay=0.0)
    _check(pair, q, see, mask=mask, causal=False)
    causal = ref.visible(n, counts, True, 0)
    _check(pair, q, see & causal, mask=mask)
    _check(pair, q, ref.visible(n, counts, True, 40), window=40)
    # the first block is the one that is hidden
    v[:32] = v[at:at + 32]
    again = Pair(1, 1, dim, 32, "int8", blocks=n // 32)
    again.append(k, v, [0], [n])
    see[:] = True
    see[::2, :32] = see[::2, at:at + 32] = False
    _check(again, q, see, mask=torch.from_numpy(see).to("cuda:0"), causal=False, decay=0.0)
    _check(again, q, see, mask=torch.from_numpy(see).to("cuda:0"), causal=False)


@pytest.mark.parametrize("counts", [1, 200])
@pytest.mark.parametrize("n,size", [(32, -1e33), (32, 1e33), (4096, -(2.0 ** 20)), (4096, 2.0 ** 20)])
def test_rows_whose_scores_are_far_from_zero(counts, n, size):
    """All scores of a row far below 0, or far above, up to where float32 still tells them apart
    to less than 1, and in one tile of any size: the result is some mean of the values, and the
    logarithm the largest score to float32's bits."""
    torch = _torch()
    _case(f"scores near {size} {counts}")
    pair = Pair(1, 1, 64, 32, "int8", blocks=n // 32)
    k = torch.zeros((n, 1, 64), device="cuda:0")
    k[:, :, 0] = 1.0
    v = _rand((n, 1, 64), "float32", 803)
    pair.append(k, v, [0], [n])
    q = torch.zeros((counts, 2, 64), device="cuda:0")
    q[..., 0] = size
    out, lse = pair.cache.attend(q, scale=1.0, return_lse=True, causal=False)
    assert torch.isfinite(out).all() and torch.isfinite(lse).all()
    held = pair.cache.read(fields=("v",))["v"][:, 0]
    slack = 2.0 ** -10 * held.abs().max()
    assert (out <= held.amax(0) + slack).all() and (out >= held.amin(0) - slack).all()
    assert ((lse.double() - size).abs() <= 8 * U * abs(size) + np.log(n)).all()
