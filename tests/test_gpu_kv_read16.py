"""What a KVCache holds, read back in 16 bits: the float32 values rounded once, whatever the
dimension, the range of slots and the alignment of the outputs, and nothing beside them."""

import ctypes
from array import array

import pytest

pytestmark = pytest.mark.gpu

DIMS = [1, 7, 8, 33, 40, 64, 72, 80, 96, 128, 160, 192, 200, 256]


def _cache(torch, dim, code, block, lens, heads):
    import vicinity_amd as va

    cache = va.KVCache(len(lens), heads, dim, sum(-(-n // block) for n in lens) + 1, block, code)
    gen = torch.Generator(device="cuda").manual_seed(dim * 8 + block)
    k, v = (torch.randn(sum(lens), heads, dim, device="cuda", generator=gen) for _ in "kv")
    cache.append(k, v, counts=lens)
    return cache


@pytest.mark.parametrize("code", ["int8", "fp8"])
@pytest.mark.parametrize("dim", DIMS)
def test_read_in_16_bits_is_the_rounded_float32(dim, code):
    import torch

    print(f"[case] read16 dim {dim} {code}", flush=True)
    lens = [1, 31, 200, 0, 333]
    cache = _cache(torch, dim, code, 64 if dim % 3 else 32, lens, 3)
    for first, counts in ((None, None), ([0, 5, 37, 0, 129], [1, 26, 101, 0, 200]), ([1, 31, 199, 0, 64], None)):
        whole = cache.read(first=first, counts=counts, fields=("k", "v"))
        for dtype in (torch.float16, torch.bfloat16):
            got = cache.read(first=first, counts=counts, dtype=dtype)
            for f in ("k", "v"):
                assert torch.equal(got[f], whole[f].to(dtype)), (f, dtype, first)
            only = cache.read(first=first, counts=counts, fields=("v",), dtype=dtype)
            assert torch.equal(only["v"], got["v"])


@pytest.mark.parametrize("offset", [0, 1, 4, 8])
@pytest.mark.parametrize("dim", [7, 64, 96, 128])
def test_outputs_of_any_alignment_and_nothing_beside_them(dim, offset):
    import torch

    from vicinity_amd import _lib

    print(f"[case] read16 dim {dim} offset {offset}", flush=True)
    lens, first, counts = [70, 150], [3, 41], [67, 90]
    cache = _cache(torch, dim, "int8", 32, lens, 2)
    whole = cache.read(first=first, counts=counts, fields=("k", "v"))
    n = sum(counts) * 2 * dim
    ptr = lambda a: a.buffer_info()[0]
    ids, at, cn = array("i", range(2)), array("q", first), array("q", counts)
    for dtype, number in ((torch.float16, 1), (torch.bfloat16, 2)):
        out = torch.full((2, offset + n + 64), 7.0, device="cuda", dtype=dtype)
        _lib.check(cache._L.vgpu_kv_read(
            cache._h, ptr(ids), ptr(at), ptr(cn), 2, number, out[0].data_ptr() + 2 * offset,
            out[1].data_ptr() + 2 * offset, None, None,
            ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)))
        torch.cuda.synchronize()
        for row, f in zip(out, ("k", "v")):
            assert torch.equal(row[offset:offset + n], whole[f].to(dtype).flatten())
            assert (row[:offset] == 7).all() and (row[offset + n:] == 7).all()
