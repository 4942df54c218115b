"""select_beams on the GPU against its definition in 64 bits.

Choices have to be equal where no two totals are closer than the kernel's error.  That error,
from the arithmetic: an exponential's argument is rounded twice (2^-23 of its size, at most
104 where it is not 0 yet; what lies below 2^-40 of the largest adds less than 2^-20 over all),
the exponential by 2^-23, and float32 sums of at most 64 of them by 2^-18: log sum is within
ERR = 2^-17 at worst, all rounding one way.  Totals are rounded once to float32."""

import numpy as np
import pytest

pytestmark = pytest.mark.gpu
ERR = 2.0 ** -17


def _case(msg):
    print(f"[case] beams: {msg}", flush=True)


def _torch():
    import torch

    return torch


def reference(logits, scores, beams, k):
    """totals, rows, tokens in float64, and all totals."""
    x = logits.detach().double().cpu().numpy()
    s = np.zeros(len(x)) if scores is None else scores.double().cpu().numpy()
    with np.errstate(invalid="ignore", divide="ignore", over="ignore"):
        top = x.max(axis=1, keepdims=True)
        shift = np.where(np.isneginf(top), 0, top)
        total = (x - shift) - np.log(np.exp(x - shift).sum(axis=1, keepdims=True))
        total = np.where(np.isneginf(top), -np.inf, s[:, None] + total)
    total[np.isneginf(s)] = -np.inf
    bad = np.isnan(x).any(axis=1) | np.isposinf(x).any(axis=1) | np.isnan(s) | np.isposinf(s)
    total[bad & ~np.isneginf(s)] = np.nan
    flat = total.reshape(len(x) // beams, beams * x.shape[1])
    key = np.where(np.isnan(flat), np.inf, flat)
    order = np.argsort(-key, axis=1, kind="stable")[:, :k]
    at = np.take_along_axis(flat, order, axis=1)
    v = x.shape[1]
    return at, order // v + beams * np.arange(len(flat))[:, None], order % v, flat


def check(logits, scores, beams, k, **kw):
    import vicinity_amd as va

    got, rows, tokens = (t.cpu().numpy() for t in va.select_beams(logits, scores, beams, k, **kw))
    want, wrows, wtokens, flat = reference(logits, scores, beams, k)
    assert got.shape == want.shape and got.dtype == np.float32
    assert rows.dtype == np.int64 and tokens.dtype == np.int64
    real = np.isfinite(want)
    assert np.array_equal(np.isnan(got), np.isnan(want))
    assert np.array_equal(np.isneginf(got), np.isneginf(want))
    err = np.abs(got[real] - want[real])
    assert (err <= ERR + 2.0 ** -24 * np.abs(want[real])).all(), err.max()
    same = (rows == wrows) & (tokens == wtokens)
    if not same.all():
        # another choice is right only where the totals are as close as the error allows
        v = logits.shape[1]
        for g, j in zip(*np.nonzero(~same)):
            mine = flat[g, (rows[g, j] - g * beams) * v + tokens[g, j]]
            assert rows[g, j] // beams == g and abs(mine - want[g, j]) <= 2 * ERR and rows[g, j] != wrows[g, j]
        picked = np.sort((rows - beams * np.arange(len(flat))[:, None]) * v + tokens, axis=1)
        assert (np.diff(picked, axis=1) > 0).all()
    return same


def inputs(groups, beams, vocab, dtype, seed=0, gain=3.0):
    torch = _torch()
    g = torch.Generator().manual_seed(seed)
    x = torch.randn((groups * beams, vocab), generator=g) * gain
    s = -10 * torch.rand((groups * beams,), generator=g)
    return x.to(getattr(torch, dtype)).to("cuda:0"), s.to("cuda:0")


@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("groups,beams,vocab,k", [
    (1, 1, 1, 1), (1, 1, 5, 5), (3, 2, 7, 9), (2, 4, 100, 8), (5, 3, 1023, 6), (1, 4, 32_000, 8),
    (2, 16, 2048, 32), (2, 16, 2049, 256), (1, 64, 4099, 128), (7, 5, 16_391, 10), (1, 1, 200_003, 256),
    (1, 1000, 333, 200), (300, 2, 50, 4), (64, 8, 20_001, 16)])
def test_against_the_definition(dtype, groups, beams, vocab, k):
    _case(f"{dtype} {groups} x {beams} x {vocab} k {k}")
    x, s = inputs(groups, beams, vocab, dtype, seed=vocab + k)
    assert check(x, s, beams, k).mean() > 0.99


@pytest.mark.parametrize("beams,k", [(1, 7), (4, 8), (8, 100)])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_without_scores_and_default_k(beams, k, dtype):
    import vicinity_amd as va

    x, _ = inputs(2, beams, 300, dtype)
    assert check(x, None, beams, k).all()
    a, b = va.select_beams(x, None, beams), va.select_beams(x, None, beams, beams)
    assert all(_torch().equal(p, q) for p, q in zip(a, b))


@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("vocab,k", [(40, 9), (5000, 40), (70_000, 256)])
def test_equal_logits_go_by_row_and_token(dtype, vocab, k):
    """Rows of one value, of two values, and equal rows: totals that are equal exactly."""
    torch = _torch()
    x = torch.zeros((4, vocab), dtype=getattr(torch, dtype), device="cuda:0")
    assert check(x, torch.zeros(4, device="cuda:0"), 4, k).all()
    x[1, vocab // 2:] = 1.0
    x[3, vocab // 2:] = 1.0
    assert check(x, torch.tensor([0.0, -1.0, 0.0, -1.0], device="cuda:0"), 4, k).all()
    x, _ = inputs(1, 1, vocab, dtype, gain=1.0)
    x = (x * 4).round() / 4  # few values
    assert check(x.expand(4, vocab), torch.full((4,), -2.0, device="cuda:0"), 4, k).all()


@pytest.mark.parametrize("dtype", ["float32", "float16"])
def test_rows_in_order(dtype):
    """Ascending and descending logits: the best of a slice lie in one place of it."""
    torch = _torch()
    for vocab, k in ((3000, 100), (40_000, 256), (66_000, 256)):
        up = torch.linspace(-8, 8, vocab, device="cuda:0").to(getattr(torch, dtype))
        x = torch.stack([up, up.flip(0), torch.roll(up, vocab // 3), up * 0.5])
        check(x, torch.tensor([-0.3, -0.1, -0.7, -0.2], device="cuda:0"), 4, k)
        check(x, None, 1, k)
        # the largest of one thread's 8 elements (4 in float32), thread after thread
        y = up.view(-1).clone()
        y[: vocab // 16 * 16] = up[: vocab // 16 * 16].view(16, -1).t().reshape(-1)
        check(y[None], None, 1, k)


@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("vocab", [50, 9000, 40_000])
def test_masked_tokens(dtype, vocab):
    torch = _torch()
    x, s = inputs(2, 4, vocab, dtype)
    x[0] = -torch.inf  # nothing can follow
    x[1, 3:] = -torch.inf  # three can
    x[2, : vocab - 2] = -torch.inf  # the last two
    x[3, torch.rand(vocab, device="cuda:0") < 0.95] = -torch.inf
    x[4:] = -torch.inf
    x[5, 17] = 0.5
    check(x, s, 4, 30)
    s[1] = -torch.inf  # a beam that has ended
    check(x, s, 4, 30)
    s[:] = -torch.inf
    check(x, s, 4, 30)
    # the least and the largest numbers of the type are numbers
    lim = torch.finfo(x.dtype)
    x, s = inputs(1, 3, vocab, dtype)
    x[0, ::2] = lim.min
    x[1] = lim.min
    x[2, 5] = lim.max
    check(x, s, 3, 20)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("vocab", [40, 30_000])
def test_what_is_not_a_number(dtype, vocab):
    torch = _torch()
    nan, inf = float("nan"), float("inf")
    for place in (0, 33, vocab - 1):
        x, s = inputs(4, 3, vocab, dtype, seed=place)
        x[1, place] = nan
        x[5, place] = inf
        x[7, :] = nan
        x[8, :] = inf
        s[9], s[10] = nan, inf
        x[11, place] = nan
        s[11] = -inf  # has ended whatever its logits are
        check(x, s, 3, 40)


@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
def test_strides_and_offsets(dtype):
    torch = _torch()
    big, s = inputs(2, 4, 20_011, dtype)
    for first in range(9):  # rows that begin at every address
        check(big[:, first:first + 5001], s, 4, 8)
    check(big[::2, 3:], s[::2], 2, 8)
    check(big[:, ::3], s, 4, 8)
    check(big.t().contiguous().t(), s, 4, 8)
    check(big[:1].expand(8, -1)[:, :3000], s, 4, 8)
    check(big[:, :1], s, 4, 4)
    check(big[:0], s[:0], 4, 4)


def test_offsets_past_32_bits():
    torch = _torch()
    vocab = 1 << 20
    x = torch.full((2200, vocab), -20.0, dtype=torch.bfloat16, device="cuda:0")  # 4.6 GB
    g = torch.Generator(device="cuda:0").manual_seed(1)
    at = torch.randint(0, vocab, (2200, 3), generator=g, device="cuda:0")
    lift = torch.rand((2200, 3), generator=g, device="cuda:0") * 8 + 4
    x.scatter_(1, at, lift.to(x.dtype))
    import vicinity_amd as va

    got, rows, tokens = va.select_beams(x, None, 2, 2)
    whole = torch.log_softmax(x[-2:].double(), dim=1).view(-1)
    best, order = torch.sort(whole, descending=True, stable=True)
    assert torch.equal(rows[-1], 2198 + order[:2] // vocab) and torch.equal(tokens[-1], order[:2] % vocab)
    assert (got[-1] - best[:2]).abs().max() <= ERR + 2.0 ** -24 * best[:2].abs().max()
    assert (rows == torch.arange(0, 2200, 2, device="cuda:0")[:, None] + rows % 2).all()


def test_the_same_answer_every_time_and_on_every_stream():
    torch = _torch()
    import vicinity_amd as va

    x, s = inputs(6, 8, 50_003, "bfloat16")
    want = va.select_beams(x, s, 8, 16)
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for i in range(6):
        st = streams[i % 2]
        got = va.select_beams(x, s, 8, 16, stream=st)
        with torch.cuda.stream(st):
            again = va.select_beams(x, s, 8, 16)
        torch.cuda.synchronize()
        for a, b, c in zip(want, got, again):
            assert torch.equal(a, b) and torch.equal(a, c)


def test_captured_into_a_graph():
    torch = _torch()
    import vicinity_amd as va

    x, s = inputs(3, 4, 9001, "float16")
    va.select_beams(x, s, 4)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = va.select_beams(x, s, 4, 8)
    for seed in range(4):  # new inputs in place, with eager work between the replays
        y, t = inputs(3, 4, 9001, "float16", seed=seed + 10)
        x.copy_(y)
        s.copy_(t)
        graph.replay()
        torch.cuda.synchronize()
        want = va.select_beams(y, t, 4, 8)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want))


def test_arguments_that_are_refused():
    torch = _torch()
    import vicinity_amd as va

    x, s = inputs(2, 2, 10, "float32")
    for args, error, match in [
            ((x, s, 3), ValueError, "rows"), ((x, s, 0), ValueError, "beams"), ((x, s, 2.0), ValueError, "beams"),
            ((x, s, 2, 21), ValueError, "k must"), ((x, s, 2, 0), ValueError, "k must"),
            ((x, s[:3], 2), ValueError, "scores"), ((x, s.double(), 2), TypeError, "scores"),
            ((x, s.cpu(), 2), ValueError, "scores"), ((x, [0.0] * 4, 2), TypeError, "scores"),
            ((x[:, :0], s, 2), ValueError, "vocab"), ((x.double(), s, 2), TypeError, "logits"),
            ((x[None], s, 2), ValueError, "logits"), ((x.cpu(), s, 2), ValueError, "logits")]:
        with pytest.raises(error, match=match):
            va.select_beams(*args)
    assert torch.equal(va.select_beams(x, s, 2)[2], va.select_beams(x, s, 2, 2)[2])
