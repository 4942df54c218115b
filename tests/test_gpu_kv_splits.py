"""Attention of few rows in more workgroups than are on the card at once, one sequence far
longer than the others: against the definitions in 64 bits."""

import pytest

from test_gpu_kv import Pair, _case, _check_attend, _rand

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,decay", [("bfloat16", None), ("bfloat16", 0.5), ("float32", None)])
@pytest.mark.parametrize("n", [110, 150])
def test_one_long_sequence_among_many(n, dtype, decay):
    _case(f"{n} sequences, one of 9000 {dtype} {decay}")
    heads, dim = 8, 32
    lens = [3 + i % 40 for i in range(n)]
    lens[n // 3] = 9000
    pair = Pair(n, heads, dim, 32, "int8", blocks=2 * n + 300)
    t = sum(lens)
    pair.append(_rand((t, heads, dim), dtype, 300, 0.7), _rand((t, heads, dim), dtype, 301), list(range(n)), lens)
    order = [(7 * i) % n for i in range(n)] if n % 7 else list(range(n))
    _check_attend(pair, _rand((n, 2 * heads, dim), dtype, 302), order, [1] * n, decay=decay)
    counts = [1 + i % 3 for i in range(n)]
    _check_attend(pair, _rand((sum(counts), 2 * heads, dim), dtype, 303), order, counts, decay=decay)
