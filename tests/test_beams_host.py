"""Selection of beams without a GPU: refusals that come before any device call, and the
struct's layout."""

import ctypes
import os
import shutil
import subprocess

import pytest

HEADER = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include",
                      "vicinity_gpu.h")


@pytest.mark.parametrize("change,match", [
    (dict(dtype=3), "dtype"), (dict(dtype=-1), "dtype"), (dict(rows=7), "rows"),
    (dict(rows=(1 << 24) + 2), "rows"), (dict(vocab=0), "vocab"), (dict(vocab=(1 << 30) + 1), "vocab"),
    (dict(beams=0), "beams"), (dict(beams=1025, rows=1025), "beams"), (dict(k=0), "k must"),
    (dict(k=257), "k must"), (dict(k=9, vocab=4), "k must"), (dict(rows=1 << 20, vocab=1 << 30), "too many"),
    (dict(rows=1024, beams=1024, vocab=1 << 27, k=256), "too many"),
    (dict(rows=1 << 22, beams=1, vocab=100), "groups")])
def test_sizes_that_are_refused(change, match):
    from vicinity_amd import _lib

    args = dict(dtype=2, rows=8, vocab=1000, beams=2, k=4) | change
    size = ctypes.c_size_t(77)
    with pytest.raises(ValueError, match=match) as e:
        _lib.check(_lib.load().vgpu_beams_workspace(args["dtype"], args["rows"], args["vocab"], args["beams"],
                                                    args["k"], ctypes.byref(size)))
    assert e.value.code == _lib.ERR_INVALID_PARAMETER and size.value == 77


@pytest.mark.parametrize("change,match", [
    (dict(logits=None), "null"), (dict(out_scores=None), "null"), (dict(out_parents=None), "null"),
    (dict(out_tokens=None), "null"), (dict(logits=4097), "inputs must be aligned"),
    (dict(scores=4098), "inputs must be aligned"), (dict(out_scores=4098), "outputs must be aligned"),
    (dict(out_parents=4100), "outputs must be aligned"), (dict(out_tokens=4100), "outputs must be aligned"),
    (dict(workspace=None), "workspace"), (dict(workspace=4104), "workspace"),
    (dict(workspace_bytes=-1), "workspace")])
def test_calls_that_are_refused(change, match):
    """(no pointer here is one that could be read)"""
    from vicinity_amd import _lib

    lib, size = _lib.load(), ctypes.c_size_t()
    _lib.check(lib.vgpu_beams_workspace(2, 8, 1000, 2, 4, ctypes.byref(size)))
    assert size.value > 8 * 4 * 8
    args = dict(logits=4096, dtype=2, stride_row=1000, stride_token=1, rows=8, vocab=1000, beams=2, k=4,
                scores=4096, stride_score=1, workspace=4096, workspace_bytes=size.value, out_scores=4096,
                out_parents=4096, out_tokens=4096) | change
    if args["workspace_bytes"] < 0:
        args["workspace_bytes"] += size.value
    with pytest.raises(ValueError, match=match):
        _lib.check(lib.vgpu_select_beams(ctypes.byref(_lib.Beams(**args)), None))


def test_null_structs_and_empty_batches():
    from vicinity_amd import _lib

    lib = _lib.load()
    assert lib.vgpu_select_beams(None, None) == _lib.ERR_INVALID_PARAMETER
    assert lib.vgpu_beams_workspace(2, 8, 1000, 2, 4, None) == _lib.ERR_INVALID_PARAMETER
    assert lib.vgpu_select_beams(ctypes.byref(_lib.Beams(dtype=2, rows=0, vocab=9, beams=2, k=1)), None) == _lib.OK


def test_tensors_that_are_refused():
    torch = pytest.importorskip("torch")
    import vicinity_amd as va

    x = torch.zeros((4, 10))
    for logits, error in ((x.numpy(), TypeError), (x.double(), TypeError), (x, ValueError), (x[0], ValueError)):
        with pytest.raises(error, match="logits"):
            va.select_beams(logits, None, 2)


def test_struct_layout_matches_the_header(tmp_path):
    from vicinity_amd import _lib

    if shutil.which("gcc") is None:
        pytest.skip("gcc not available")
    body = [f'#include <stdio.h>\n#include <stddef.h>\n#include "{HEADER}"\nint main(void) {{',
            'printf("size %zu\\n", sizeof(vgpu_beams));']
    body += [f'printf("{f} %zu\\n", offsetof(vgpu_beams, {f}));' for f, _ in _lib.Beams._fields_]
    src, exe = tmp_path / "probe.c", tmp_path / "probe"
    src.write_text("\n".join(body + ["return 0; }"]))
    subprocess.run(["gcc", "-std=c11", "-o", str(exe), str(src)], check=True)
    out = subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout
    got = dict(line.split() for line in out.splitlines())
    assert int(got.pop("size")) == ctypes.sizeof(_lib.Beams)
    assert {f: int(v) for f, v in got.items()} == {f: getattr(_lib.Beams, f).offset for f, _ in _lib.Beams._fields_}
