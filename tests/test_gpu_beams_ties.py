"""select_beams where float64 holds the totals of different logits as equal: a score so low that
it swallows the logits (a beam that was never begun has the type's least score), logits that lie
closer together than float64 tells beside the row's logarithm.  By the definition the larger
logit still has the larger total, so a row's tokens come in the order of their logits, of equal
ones the lower token; between rows with equal totals the lower row comes first."""

import numpy as np
import pytest

from test_gpu_beams import inputs

pytestmark = pytest.mark.gpu


def _case(msg):
    print(f"[case] beams, totals that float64 holds as equal: {msg}", flush=True)


def _order(x, k):
    """Tokens of the k largest logits of each row."""
    return np.argsort(-x.double().cpu().numpy(), axis=1, kind="stable")[:, :k]


@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("score", [-1e30, float(np.finfo(np.float32).min)])
@pytest.mark.parametrize("beams,vocab,k", [(1, 37, 9), (1, 50_021, 5), (4, 20_001, 16), (3, 70_001, 256), (64, 3001, 100)])
def test_scores_that_swallow_the_logits(dtype, score, beams, vocab, k):
    import torch

    import vicinity_amd as va

    _case(f"{dtype} score {score} {beams} x {vocab} k {k}")
    x, _ = inputs(2, beams, vocab, dtype, seed=k)
    s = torch.full((2 * beams,), score, device="cuda:0")
    totals, rows, tokens = va.select_beams(x, s, beams, k)
    want = _order(x, k)[::beams]  # the first row of each group has vocab >= k tokens
    assert torch.equal(totals, torch.full_like(totals, score))
    assert (rows == torch.tensor([[0], [beams]], device="cuda:0")).all()
    assert np.array_equal(tokens.cpu().numpy(), want)
    if beams > 1:  # a beam that was begun, beside them
        s[beams - 1] = -1.0
        totals, rows, tokens = va.select_beams(x, s, beams, k)
        first = min(k, vocab)
        assert rows[0, :first].tolist() == [beams - 1] * first
        assert np.array_equal(tokens[0, :first].cpu().numpy(), _order(x[beams - 1:beams], first)[0])


@pytest.mark.parametrize("vocab,k", [(100, 12), (30_011, 64)])
def test_logits_closer_than_float64_tells(vocab, k):
    import torch

    import vicinity_amd as va

    _case(f"{vocab} k {k}")
    g = torch.Generator().manual_seed(k)
    x = torch.full((2, vocab), -9.0)
    at = torch.randperm(vocab, generator=g)[:80]
    x[0, at] = torch.randperm(80, generator=g).float() * 1e-25  # beside log(80): one number in float64
    x[1] = x[0].flip(0)
    x = x.to("cuda:0")
    totals, rows, tokens = va.select_beams(x, None, 1, k)
    assert (totals == totals[0, 0]).all()
    assert np.array_equal(tokens.cpu().numpy(), _order(x, k))
    # of two rows with equal totals the lower one's tokens come first
    y = torch.cat([x[1:], x[1:]])
    totals, rows, tokens = va.select_beams(y, None, 2, k)
    assert (rows == 0).all() and np.array_equal(tokens.cpu().numpy(), _order(x[1:], k))


def test_more_equal_totals_than_are_put_in_order_at_once():
    """Every entry of 64 rows' lists has one total: the k best are kept through pieces of them."""
    import torch

    import vicinity_amd as va

    x, _ = inputs(1, 64, 9001, "float32", seed=3)
    s = torch.full((64,), -3e38, device="cuda:0")
    totals, rows, tokens = va.select_beams(x, s, 64, 256)
    assert (rows == 0).all() and np.array_equal(tokens.cpu().numpy(), _order(x[:1], 256))
    x[0] = -torch.inf  # no token can follow the first: its totals come last
    totals, rows, tokens = va.select_beams(x, s, 64, 256)
    assert (rows == 1).all() and np.array_equal(tokens.cpu().numpy(), _order(x[1:2], 256))
