"""The build of the C library beside the binding that needs torch (a library of one
small source; nvcc needs no GPU)."""
import os
import subprocess
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def run(tmp_path, before="", after=""):
    for d in ("csrc/python", "include", "out", "build"):
        os.makedirs(tmp_path / d, exist_ok=True)
    if not (tmp_path / "csrc" / "lib.cpp").exists():
        (tmp_path / "csrc" / "lib.cpp").write_text('extern "C" int answer() { return 7; }\n')
        (tmp_path / "csrc" / "python" / "ext.cpp").write_text("int nothing() { return 0; }\n")
        (tmp_path / "include" / "lib.h").write_text("int answer();\n")
    code = f"""
import os, sys
{before}
from laya_goish_b200 import build
t = {str(tmp_path)!r}
build.PKG, build.CSRC, build.INCLUDE, build.BUILD = t + "/out", t + "/csrc", t + "/include", t + "/build"
build.OUT, build.EXT_OUT = t + "/out/liblaya_cuda.so", t + "/out/_device.so"
build.EXT_SRC = t + "/csrc/python/ext.cpp"
{after}
build.build()
"""
    return subprocess.run([sys.executable, "-c", code], cwd=ROOT, capture_output=True, text=True)


@pytest.mark.parametrize("gone", ["torch is not installed", "the binding does not compile"])
def test_the_library_needs_no_binding(tmp_path, gone):
    if gone.startswith("torch"):
        r = run(tmp_path, before="sys.modules['torch'] = None")
        assert r.returncode == 0, r.stderr
        assert "_device.so is not built" in r.stderr
    else:
        os.makedirs(tmp_path / "csrc" / "python")
        r = run(tmp_path, after="open(build.EXT_SRC, 'w').write('int nothing( {')")
        assert r.returncode != 0 and "g++ failed" in r.stderr
    assert (tmp_path / "out" / "liblaya_cuda.so").exists() and not (tmp_path / "out" / "_device.so").exists()


def test_the_binding_is_built_again_for_another_torch(tmp_path):
    obj = tmp_path / "build" / "device_ext.o"
    times = []
    for version in ("", "", "importlib.metadata.version = lambda name: '99.0'", ""):
        r = run(tmp_path, after="import importlib.metadata\n" + version)
        assert r.returncode == 0, r.stderr
        times.append(obj.stat().st_mtime_ns)
    assert times[0] == times[1] < times[2] < times[3]
    assert (tmp_path / "out" / "_device.so").exists()
