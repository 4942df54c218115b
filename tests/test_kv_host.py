"""The attention memory without a GPU: refusals that come before any device call, struct
layouts, and the numpy definitions that the GPU tests compare with."""

import ctypes
import os
import shutil
import subprocess

import kv_reference as ref
import numpy as np
import pytest

HEADER = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include",
                      "vicinity_gpu.h")


@pytest.mark.parametrize("change,match", [
    (dict(num_seqs=0), "num_seqs"), (dict(num_heads=0), "num_heads"), (dict(head_dim=0), "head_dim"),
    (dict(head_dim=257), "head_dim"), (dict(num_blocks=0), "num_blocks"),
    (dict(block_tokens=16), "block_tokens"), (dict(block_tokens=65), "block_tokens"),
    (dict(code=2), "code"), (dict(num_blocks=1 << 30), "slots"), (dict(num_heads=1 << 40), "num_heads")])
def test_new_refuses_impossible_caches(change, match):
    from vicinity_amd import _lib

    args = dict(num_seqs=1, num_heads=1, head_dim=64, num_blocks=1, block_tokens=32, max_blocks=0,
                code=0) | change
    h = ctypes.c_void_p()
    with pytest.raises(ValueError, match=match) as e:
        _lib.check(_lib.load().vgpu_kv_new(ctypes.byref(_lib.KvParams(**args)), ctypes.byref(h)))
    assert e.value.code == _lib.ERR_INVALID_CONFIG and not h.value


def test_null_handles_are_refused():
    from vicinity_amd import _lib

    lib = _lib.load()
    x, q = _lib.KvTensor(), _lib.KvQuery()
    calls = [lambda: lib.vgpu_kv_new(None, None), lambda: lib.vgpu_kv_get_info(None, None),
             lambda: lib.vgpu_kv_lengths(None, None),
             lambda: lib.vgpu_kv_append(None, None, None, 0, ctypes.byref(x), ctypes.byref(x), None, None, None),
             lambda: lib.vgpu_kv_attend(None, None, None, 0, ctypes.byref(q), None),
             lambda: lib.vgpu_kv_evict(None, None, None, 0, 0, 0, 0, None, None, None, None),
             lambda: lib.vgpu_kv_read(None, None, None, None, 0, 0, None, None, None, None, None),
             lambda: lib.vgpu_kv_truncate(None, None, None, 0)]
    for call in calls:
        assert call() == _lib.ERR_INVALID_PARAMETER
    lib.vgpu_kv_free(None)


def test_struct_layouts_match_the_header(tmp_path):
    from vicinity_amd import _lib

    if shutil.which("gcc") is None:
        pytest.skip("gcc not available")
    structs = {"vgpu_kv_params": _lib.KvParams, "vgpu_kv_info": _lib.KvInfo, "vgpu_tensor3": _lib.KvTensor,
               "vgpu_kv_query": _lib.KvQuery}
    body = [f'#include <stdio.h>\n#include <stddef.h>\n#include "{HEADER}"\nint main(void) {{']
    for name, py in structs.items():
        body.append(f'printf("{name} size %zu\\n", sizeof({name}));')
        body += [f'printf("{name} {f} %zu\\n", offsetof({name}, {f}));' for f, _ in py._fields_]
    src, exe = tmp_path / "probe.c", tmp_path / "probe"
    src.write_text("\n".join(body + ["return 0; }"]))
    subprocess.run(["gcc", "-std=c11", "-o", str(exe), str(src)], check=True)
    out = subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout
    got = {tuple(line.split()[:2]): int(line.split()[2]) for line in out.splitlines()}
    for name, py in structs.items():
        assert got[(name, "size")] == ctypes.sizeof(py)
        for f, _ in py._fields_:
            assert got[(name, f)] == getattr(py, f).offset, (name, f)


def test_e4m3_reference_against_torch():
    torch = pytest.importorskip("torch")
    x = np.concatenate([np.linspace(-448, 448, 200_001), np.geomspace(1e-4, 448, 50_000)]).astype(np.float32)
    x = np.concatenate([x, ((ref.E4M3[1:] + ref.E4M3[:-1]) / 2).astype(np.float32)])  # the ties
    want = torch.from_numpy(x).to(torch.float8_e4m3fn).float().numpy()
    assert np.array_equal(ref.to_e4m3(x), want)


@pytest.mark.parametrize("code", ["int8", "fp8"])
def test_stored_values_are_within_half_a_step(code):
    rng = np.random.default_rng(1)
    st = ref.Store(2, 16, 32, code)
    x = rng.standard_normal((100, 2, 16)).astype(np.float32)
    for part in np.split(x, [1, 40, 41, 90]):
        st.append(part)
    # one rounding, and one more for each time that the block's scale grew: at most the
    # pieces that enter one block (3 here) and half a step of the last scale each
    s = np.repeat(st.scales, 32, axis=0)[:100, :, None]
    step = s if code == "int8" else np.maximum(np.abs(st.values()) / 8, s * 2.0 ** -9)
    assert (np.abs(st.values() - x) <= 3 * 0.5 * step * 1.2).all()


def test_attention_reference_by_hand():
    k = np.array([[[1.0, 0.0]], [[0.0, 1.0]], [[0.0, 0.0]]])
    v = np.array([[[1.0, 2.0]], [[3.0, 4.0]], [[5.0, 6.0]]])
    q = np.array([[[np.log(2.0), 0.0]], [[0.0, np.log(3.0)]]])
    out, lse, w = ref.attend(q, k, v, ref.visible(3, 2, True, 0), 1.0)
    # token 0 stands at slot 1: weights 2, 1; token 1 at slot 2: weights 1, 3, 1
    assert np.allclose(out[0, 0], (2 * v[0, 0] + v[1, 0]) / 3)
    assert np.allclose(out[1, 0], (v[0, 0] + 3 * v[1, 0] + v[2, 0]) / 5)
    assert np.allclose(lse[:, 0], np.log([3.0, 5.0]))
    assert np.allclose(w[:, 0], [2 / 3 + 1 / 5, 1 / 3 + 3 / 5, 1 / 5])
    assert ref.visible(3, 2, True, 1).tolist() == [[False, True, False], [False, False, True]]
    assert not ref.visible(1, 3, True, 0)[:2].any()


def test_keep_slots_ties_and_recent():
    w = np.array([1.0, 3.0, 1.0, 0.0, np.nan, 1.0, 9.0])[:, None]
    stay, gone = ref.keep_slots(w, 4, 1)
    assert stay[:, 0].tolist() == [0, 1, 4, 6] and gone[:, 0].tolist() == [2, 3, 5]
    stay, gone = ref.keep_slots(w, 7, 2)
    assert stay[:, 0].tolist() == list(range(7)) and gone.shape == (0, 1)
