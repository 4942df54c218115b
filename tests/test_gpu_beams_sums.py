"""select_beams adds a row's exponentials in float64, as it says: rows whose sums differ by less
than float32 sums can hold are still told apart.

Terms of 1 and of s = 2^-25: a float32 sum that has reached 1 loses each of the small ones (half a
unit in the last place of 1 is 2^-24), a float64 sum holds all.  Row a has a one at every W-th
token, where the 16 bytes begin that a thread loads at once, and small terms else: m ones and n
small terms, m + n s.  Row b has the same ones and a single term of about n s / 2.  As
m < sum of b < sum of a, the best token of b comes first; where small terms are lost, a's does.

The exponentials of 0 are exact.  A small one's argument, up to 25 in base 2, is rounded by 2^-20
and the constant log2 e by 2^-26 of itself, so it is off by less than 2^-19 of itself."""

import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu


def _case(msg):
    print(f"[case] beams' sums: {msg}", flush=True)


@pytest.mark.parametrize("dtype,w", [("float32", 4), ("float16", 8), ("bfloat16", 8)])
@pytest.mark.parametrize("vocab", [1024, 16_384, 100_000])
def test_small_terms_beside_large_ones(dtype, w, vocab):
    import torch

    import vicinity_amd as va

    _case(f"{dtype} vocab {vocab}")
    t = getattr(torch, dtype)
    small = torch.tensor(-25 * math.log(2), dtype=t)
    s = math.exp(float(small.double()))
    a = torch.full((vocab,), float(small), dtype=t)
    a[::w] = 0.0
    m = int((a == 0).sum())
    sum_a = m + (vocab - m) * s
    # b: the same ones, and one term that makes half of what a's small ones add
    b = torch.full((vocab,), -math.inf, dtype=t)
    b[::w] = 0.0
    b[1] = math.log((vocab - m) * s / 2)
    sum_b = m + math.exp(float(b[1].double()))
    assert m < sum_b < sum_a
    for rows in ((a, b), (b, a)):
        x = torch.stack(rows).to("cuda:0")
        totals, parents, tokens = va.select_beams(x, None, 2, 2)
        want = int(rows[1] is b)  # b's totals are the larger ones
        assert parents.tolist() == [[want, want]] and tokens.tolist() == [[0, w]]
        # the total itself: float64, then one rounding to float32
        err = abs(float(totals[0, 0].double()) + math.log(sum_b))
        assert err <= 2.0 ** -24 * math.log(sum_b) + 2.0 ** -40 + (sum_b - m) / m * 2.0 ** -19, err
        one = va.select_beams(x[1 - want:2 - want].contiguous(), None, 1, 1)[0]
        err = abs(float(one[0, 0].double()) + math.log(sum_a))
        assert err <= 2.0 ** -24 * math.log(sum_a) + 2.0 ** -40 + (sum_a - m) / m * 2.0 ** -19, err


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_sums_near_the_exact_ones(dtype):
    """Ordinary rows.  Of a term e^-y the exponential's argument is rounded twice, by 2^-24 of
    y log2 e and of the product, and the exponential by 2^-23: the sum is off by at most the mean
    of 2^-22 (1 + y) over the terms' shares, all rounding one way."""
    import torch

    import vicinity_amd as va

    g = torch.Generator().manual_seed(5)
    for vocab in (777, 50_021):
        x = (torch.randn((24, vocab), generator=g) * 3).to(getattr(torch, dtype))
        y = x.double().numpy()
        top = y.max(axis=1, keepdims=True)
        e = np.exp(y - top)
        share = e / e.sum(axis=1, keepdims=True)
        bound = 2.0 ** -22 * (share * (1 + top - y)).sum(axis=1)
        want = -np.log(e.sum(axis=1))
        got = va.select_beams(x.to("cuda:0"), None, 1, 1)[0].cpu().double().numpy()[:, 0]
        assert (np.abs(got - want) <= bound + 2.0 ** -24 * np.abs(want)).all()
