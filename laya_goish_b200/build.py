"""Builds liblaya_cuda.so in-tree for sm_100a (nvcc cross-compiles without a GPU),
and, where torch is installed, _device.so, the Python binding of the operators
on torch tensors.

    python -m laya_goish_b200.build          # incremental
    python -m laya_goish_b200.build --clean  # full rebuild
"""
from __future__ import annotations

import concurrent.futures as cf
import glob
import importlib.metadata
import importlib.util
import os
import shutil
import subprocess
import sys
import sysconfig

PKG = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(PKG)
CSRC = os.path.join(PKG, "csrc")
INCLUDE = os.path.join(ROOT, "include")
OUT = os.path.join(PKG, "liblaya_cuda.so")
EXT_SRC = os.path.join(CSRC, "python", "device_ext.cpp")
EXT_OUT = os.path.join(PKG, "_device.so")
BUILD = os.path.join(PKG, "_build")
ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]
NVCC = os.environ.get("NVCC", "/usr/local/cuda/bin/nvcc" if os.path.exists("/usr/local/cuda/bin/nvcc") else "nvcc")
FLAGS = ["-O3", "-std=c++17", "-lineinfo", "-Xcompiler", "-fPIC", "-I", CSRC, "-I", INCLUDE]


def _sources():
    return sorted(glob.glob(os.path.join(CSRC, "*.cu")) + glob.glob(os.path.join(CSRC, "*.cpp")))


def _headers():
    return glob.glob(os.path.join(CSRC, "*.h")) + glob.glob(os.path.join(CSRC, "*.cuh")) + glob.glob(os.path.join(INCLUDE, "*.h"))


def _compile(src: str) -> str:
    obj = os.path.join(BUILD, os.path.basename(src) + ".o")
    newest_dep = max([os.path.getmtime(src)] + [os.path.getmtime(h) for h in _headers()])
    if os.path.exists(obj) and os.path.getmtime(obj) >= newest_dep:
        return obj
    cmd = [NVCC, *ARCH, *FLAGS, "-c", src, "-o", obj]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"nvcc failed for {src}:\n{r.stdout}\n{r.stderr}")
    return obj


def _compile_ext() -> str | None:
    """The binding's object file (torch's headers, the host compiler); None
    without torch, for which there is nothing to bind.  Built again for another
    torch or Python, whose ABI may differ."""
    if importlib.util.find_spec("torch") is None:
        print("torch is not installed: _device.so is not built", file=sys.stderr)
        return None
    obj, stamp = os.path.join(BUILD, "device_ext.o"), os.path.join(BUILD, "device_ext.for")
    try:
        version = importlib.metadata.version("torch")
    except importlib.metadata.PackageNotFoundError:  # a source tree on the path
        version = "of unknown version"
    built_for = f"torch {version} {importlib.util.find_spec('torch').origin}\n{sys.version}\n"
    newest = max(os.path.getmtime(f) for f in [EXT_SRC] + glob.glob(os.path.join(INCLUDE, "*.h")))
    if os.path.exists(obj) and os.path.getmtime(obj) >= newest and os.path.exists(stamp):
        with open(stamp) as f:
            if f.read() == built_for:
                return obj
    import torch
    from torch.utils import cpp_extension

    cuda = os.path.dirname(os.path.dirname(NVCC)) if os.path.isabs(NVCC) else "/usr/local/cuda"
    dirs = [INCLUDE, sysconfig.get_paths()["include"], os.path.join(cuda, "include"), *cpp_extension.include_paths()]
    cmd = [os.environ.get("CXX", "g++"), "-O2", "-std=c++17", "-fPIC", "-w",
           f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}", *[f"-I{d}" for d in dirs], "-c", EXT_SRC,
           "-o", obj]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"g++ failed for {EXT_SRC}:\n{r.stdout}\n{r.stderr}")
    with open(stamp, "w") as f:
        f.write(built_for)
    return obj


def _link_ext(obj: str) -> None:
    if os.path.exists(EXT_OUT) and os.path.getmtime(EXT_OUT) >= os.path.getmtime(obj):
        return
    from torch.utils import cpp_extension

    libs = [f"-L{d}" for d in cpp_extension.library_paths()]
    cmd = [os.environ.get("CXX", "g++"), "-shared", "-o", EXT_OUT + ".tmp", obj, f"-L{PKG}", "-l:liblaya_cuda.so",
           "-Wl,-rpath,$ORIGIN", *libs, "-lc10", "-lc10_cuda", "-ltorch_cpu", "-ltorch", "-ltorch_python"]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"link failed:\n{r.stdout}\n{r.stderr}")
    os.replace(EXT_OUT + ".tmp", EXT_OUT)


def build(clean: bool = False) -> str:
    if clean and os.path.isdir(BUILD):
        shutil.rmtree(BUILD)
    os.makedirs(BUILD, exist_ok=True)
    with cf.ThreadPoolExecutor(max_workers=min(8, os.cpu_count() or 4)) as ex:
        ext = ex.submit(_compile_ext)
        objs = list(ex.map(_compile, _sources()))
        if not os.path.exists(OUT) or os.path.getmtime(OUT) < max(os.path.getmtime(o) for o in objs):
            cmd = [NVCC, *ARCH, "-shared", "-o", OUT + ".tmp", *objs, "-lpthread"]
            r = subprocess.run(cmd, capture_output=True, text=True)
            if r.returncode != 0:
                raise RuntimeError(f"link failed:\n{r.stdout}\n{r.stderr}")
            os.replace(OUT + ".tmp", OUT)
    # the library is there whether or not the binding can be
    if ext_obj := ext.result():
        _link_ext(ext_obj)
    return OUT


if __name__ == "__main__":
    print(build(clean="--clean" in sys.argv))
