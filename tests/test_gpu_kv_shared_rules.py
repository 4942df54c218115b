"""Which way attention of forks goes: by 16 rows, by many rows, or each sequence by itself; around
the sizes where that changes, against the definition in 64 bits."""

import numpy as np
import pytest

from test_gpu_kv import _rand
from test_gpu_kv_shared import _check_large, _large

pytestmark = pytest.mark.gpu


def _case(msg):
    print(f"[case] kv shared rules: {msg}", flush=True)


# forks, query heads to a head, slots: (forks * group / 16) * 8 heads * slots / 32 tiles of 16 rows
@pytest.mark.parametrize("dim,dtype", [(64, "bfloat16"), (64, "float32"), (96, "float16"), (128, "bfloat16"),
                                       (128, "float32"), (192, "bfloat16"), (192, "float32"), (256, "float16")])
@pytest.mark.parametrize("forks,group,slots", [(61, 4, 16_352), (61, 4, 16_384), (37, 7, 33_000)])
def test_around_the_tiles_of_the_kernel_of_many_rows(dim, dtype, forks, group, slots):
    _case(f"{dim} {dtype} {forks} x {group} rows over {slots}")
    cache = _large(slots, [5 + i % 3 for i in range(forks)], 8, dim, 64, "int8", dtype)
    q = _rand((forks, 8 * group, dim), dtype, 7)
    _check_large(cache, q, list(range(1, forks + 1)), [1] * forks)
