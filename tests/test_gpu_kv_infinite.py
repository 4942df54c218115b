"""Queries with an infinite element: NaN for the rows that see a slot, whatever the scores'
signs, and nothing of it in other rows: those are as near to the exact result as without it
(the bounds of the attention's own tests; their bits may differ, since a wave moves the
references of all its rows where one row's score asks for it)."""

import numpy as np
import pytest

from test_gpu_kv import OUT_EPS, U, Pair, _case, _rand, _torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["bfloat16", "float16", "float32"])
@pytest.mark.parametrize("n,counts", [(70, 1), (70, 90), (5000, 1), (5000, 260)])
@pytest.mark.parametrize("sign", [1, -1])
def test_an_infinite_query_element_is_not_a_row_without_slots(dtype, n, counts, sign):
    """Every key's element has the same sign there, so that all scores are -inf, or inf."""
    torch = _torch()
    _case(f"infinite query {dtype} {n} {counts} {sign}")
    heads, group, dim = 2, 2, 64
    pair = Pair(1, heads, dim, 64, "int8", blocks=100)
    k, v = _rand((n, heads, dim), dtype, 700, 0.5), _rand((n, heads, dim), dtype, 701)
    k[:, :, 9] = -2.0
    pair.cache.append(k, v)
    q = _rand((counts, heads * group, dim), dtype, 702)
    held = pair.cache.read(fields=("k", "v"))
    top = float((held["k"].abs().amax(0).repeat_interleave(group, 0) * q.float().abs().amax(0)).sum(1).max())
    e = (dim + 16) * U * (top / np.sqrt(dim) + 32)
    rel = 2 * e + (2.0 ** -22 if dtype == "float32" else 2.0 ** -11) + n * (2 * U + 2.0 ** -30)
    vmax = float(held["v"].abs().max())
    bad = q.clone()
    bad[-1, 1, 9] = sign * float("inf")  # the last token, a query head of head 0
    for decay in (None, 0.0):
        want, want_lse = pair.cache.attend(q, decay=decay, return_lse=True)
        want_w = pair.cache.read(fields=("weights",))["weights"]
        out, lse = pair.cache.attend(bad, decay=decay, return_lse=True)
        assert torch.isnan(out[-1, 1]).all() and torch.isnan(lse[-1, 1])
        out[-1, 1], lse[-1, 1] = want[-1, 1], want_lse[-1, 1]
        limit = vmax * rel + OUT_EPS[dtype] * (want.double().abs() + 2 * vmax * rel)
        assert ((out.double() - want.double()).abs() <= 2 * limit).all()
        empty = torch.isneginf(want_lse)  # (90 tokens of 70 slots: the first see nothing)
        assert torch.equal(torch.isneginf(lse), empty)
        got, ref = lse[~empty].double(), want_lse[~empty].double()
        assert ((got - ref).abs() <= 2 * (2 * e + n * 2 * U + 4 * U * ref.abs())).all()
    w = pair.cache.read(fields=("weights",))["weights"]
    rows = counts * group
    assert torch.isnan(w[:, 0]).all()
    limit = (3 * e + (n + rows + 8) * 2 * U) * want_w[:, 1].double() + rows * 2.0 ** -100
    assert ((w[:, 1].double() - want_w[:, 1].double()).abs() <= 2 * limit).all()
    # a row that sees nothing still gets 0
    mask = torch.ones((counts, n), dtype=torch.bool, device="cuda:0")
    mask[-1] = False
    out, lse = pair.cache.attend(bad, mask=mask, decay=0.0, return_lse=True)
    assert not out[-1].any() and torch.isneginf(lse[-1]).all() and torch.isfinite(out).all()
    assert torch.isfinite(pair.cache.read(fields=("weights",))["weights"]).all()
