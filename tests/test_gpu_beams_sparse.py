"""select_beams where a grammar leaves few tokens: slices with fewer numbers than results, slices of
-inf alone, and around the sizes of a slice's list (1024 tokens) and of its pieces (512)."""

import numpy as np
import pytest

from test_gpu_beams import check, inputs

pytestmark = pytest.mark.gpu


def _case(msg):
    print(f"[case] beams, few tokens: {msg}", flush=True)


def _torch():
    import torch

    return torch


@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("allowed", [0, 1, 7, 40, 300, 1000, 1023, 1024, 1025, 2500])
def test_numbers_of_allowed_tokens(dtype, allowed):
    torch = _torch()
    vocab, k = 50_021, 40
    _case(f"{dtype} {allowed} of {vocab}")
    rng = np.random.default_rng(allowed)
    x, s = inputs(2, 4, vocab, dtype, seed=allowed)
    hide = torch.ones_like(x, dtype=torch.bool)
    for row in range(8):
        hide[row, torch.from_numpy(rng.permutation(vocab)[:allowed]).to(x.device)] = False
    x[hide] = -torch.inf
    check(x, s, 4, k)
    # one behind the other: all in one slice, within few threads
    for first in (0, 3, 16_380, vocab - allowed):
        y, s = inputs(1, 3, vocab, dtype, seed=first + 1)
        y[:, :first] = -torch.inf
        y[:, first + allowed:] = -torch.inf
        check(y, s, 3, k)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("vocab,k", [(30, 30), (300, 256), (1500, 256), (20_000, 256)])
def test_more_results_than_allowed_tokens(dtype, vocab, k):
    """-inf follows in the order of the tokens, also where other rows have numbers left."""
    torch = _torch()
    x, s = inputs(2, 2, vocab, dtype)
    x[torch.rand((4, vocab), device="cuda:0") < 0.99] = -torch.inf
    check(x, s, 2, k)
    x[1] = -torch.inf
    x[3, 1:] = -torch.inf
    check(x, s, 2, k)


@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
def test_the_least_number_is_a_number(dtype):
    """Beside -inf the type's least number is a token that can follow."""
    torch = _torch()
    vocab = 20_000
    x = torch.full((4, vocab), -torch.inf, dtype=getattr(torch, dtype), device="cuda:0")
    low = torch.finfo(x.dtype).min
    x[0, 5::97] = low
    x[1, 5::7] = low
    x[2, 100:110] = low
    x[2, 109] = 1.0
    x[3] = low
    check(x, None, 1, 30)
    check(x[3:], None, 1, 256)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_nan_among_few_numbers(dtype):
    """A row with NaN has totals of NaN alone, whatever its other tokens are; of many NaN none
    may take the places of the list."""
    torch = _torch()
    vocab = 40_000
    for many in (1, 600, 5000, vocab):
        x, s = inputs(1, 4, vocab, dtype)
        x[:, 50:] = -torch.inf
        x[1, vocab - many:] = float("nan")
        x[2] = 0.0
        x[2, : min(many, vocab - 1)] = float("nan")
        x[3] = 0.0
        x[3, :min(many, vocab - 1)] = -float("nan")
        check(x, s, 4, 200)
        check(x, s, 1, 200)


def test_few_tokens_take_no_longer_than_many():
    """A strict grammar is an ordinary call: 31 passes over the rows, one for each bit of a key,
    took 16 times as long.  (Medians; 4 times as long is far off either.)"""
    torch = _torch()
    import vicinity_amd as va

    x, s = inputs(32, 8, 100_003, "bfloat16")

    def median(y):
        times = []
        for _ in range(15):
            a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            a.record()
            for _ in range(5):
                va.select_beams(y, s, 8, 16)
            b.record()
            b.synchronize()
            times.append(a.elapsed_time(b))
        return sorted(times)[7]

    dense = median(x)
    for allowed in (0, 5, 40, 300):
        y = x.clone()
        y[torch.rand(y.shape, device="cuda:0") >= allowed / y.shape[1]] = -torch.inf
        took = median(y)
        _case(f"{allowed} allowed {took / 5e-3:.1f} us, all {dense / 5e-3:.1f} us")
        assert took <= 4 * dense
