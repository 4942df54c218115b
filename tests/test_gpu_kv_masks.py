"""Masks in the kernel of many rows and in the second pass that makes weights, at every padded
head dimension, against the definitions in 64 bits."""

import pytest

from test_gpu_kv import Pair, _case, _check_attend, _rand, _torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("code", ["int8", "fp8"])
@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
@pytest.mark.parametrize("dim", [33, 96, 128, 136, 192, 256])
def test_masks_of_many_rows(code, dtype, dim):
    """Rows without a slot, tiles without one, a window, weights and none."""
    torch = _torch()
    n, counts, heads, group = [2500, 700], [300, 90], 2, 4
    _case(f"masks of many rows {code} {dtype} dim {dim}")
    pair = Pair(2, heads, dim, 64, code, blocks=64)
    t = sum(n)
    pair.append(_rand((t, heads, dim), dtype, 600, 0.7), _rand((t, heads, dim), dtype, 601), [0, 1], n)
    g = torch.Generator().manual_seed(602)
    mask = torch.rand((sum(counts), max(n)), generator=g) < 0.4
    mask[5] = mask[299] = mask[310:340] = False
    mask[:, 512:640] = False
    mask = mask.to("cuda:0")
    q = _rand((sum(counts), heads * group, dim), dtype, 603)
    _check_attend(pair, q, [0, 1], counts, mask=mask)
    _check_attend(pair, q, [0, 1], counts, mask=mask, decay=0.5, causal=False)
    _check_attend(pair, q, [0, 1], counts, mask=mask, decay=1.0, window=400)
