"""In-tree build of libb2blas.so (sm_100a only) with nvcc.

``python -m hpcdeepneuralnetworks_b200.build`` compiles every ``csrc/*.cu`` into objects under
``csrc/build/`` (skipping files whose object is newer than all sources/headers) and links
``hpcdeepneuralnetworks_b200/libb2blas.so``, then the C++ driver and, where there is a torch for CUDA, the Python
extension that shortens the calls of ``layer.py`` (``csrc/calls.cpp``).  nvcc cross-compiles without a GPU.
"""
from __future__ import annotations

import glob
import importlib.util
import os
import re
import shutil
import subprocess
import sys
import sysconfig
from concurrent.futures import ThreadPoolExecutor

PKG = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(PKG, "csrc")
OBJ = os.path.join(CSRC, "build")
LIB = os.path.join(PKG, "libb2blas.so")

NVCC_FLAGS = [
    "-gencode", "arch=compute_100a,code=sm_100a", "-lineinfo", "-O3", "-std=c++17",
    "-Xcompiler", "-fPIC", "--expt-relaxed-constexpr", "-cudart", "shared",
]


def nvcc() -> str:
    exe = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    if not os.path.exists(exe):
        raise RuntimeError("nvcc not found: the CUDA kernels cannot be built")
    return exe


def _stale(target: str, deps: list[str]) -> bool:
    if not os.path.exists(target):
        return True
    t = os.path.getmtime(target)
    return any(os.path.getmtime(d) > t for d in deps)


def build(verbose: bool = False, force: bool = False, ptxas_info: bool = False) -> str:
    os.makedirs(OBJ, exist_ok=True)
    sources = sorted(glob.glob(os.path.join(CSRC, "*.cu")))
    headers = sorted(glob.glob(os.path.join(CSRC, "*.cuh"))) + sorted(glob.glob(os.path.join(CSRC, "*.inc"))) + [os.path.join(PKG, "..", "include", "b2blas.h")]
    jobs = []
    objs = []
    for src in sources:
        obj = os.path.join(OBJ, os.path.basename(src)[:-3] + ".o")
        objs.append(obj)
        if force or _stale(obj, [src] + headers):
            cmd = [nvcc()] + NVCC_FLAGS + (["-Xptxas", "-v"] if ptxas_info else []) + ["-c", src, "-o", obj]
            jobs.append(cmd)

    def run(cmd):
        r = subprocess.run(cmd, capture_output=True, text=True)
        if r.returncode != 0:
            raise RuntimeError("nvcc failed:\n" + " ".join(cmd) + "\n" + r.stdout + r.stderr)
        return r.stdout + r.stderr

    if jobs:
        with ThreadPoolExecutor(max_workers=min(8, len(jobs))) as ex:
            for out in ex.map(run, jobs):
                if verbose or ptxas_info:
                    sys.stderr.write(out)
    if jobs or force or _stale(LIB, objs):
        cmd = [nvcc(), "-shared", "-cudart", "shared", "-o", LIB] + objs + \
              ["-Xlinker", "-rpath,/usr/local/cuda/lib64", "-ldl"]
        run(cmd)
    build_driver()
    build_calls(force)
    return LIB


DRIVER_SRC = os.path.join(PKG, "drivers", "b2_driver.cpp")
DRIVER_BIN = os.path.join(PKG, "drivers", "b2_driver")


def build_driver() -> str:
    """The C++ command-line driver (reference-shaped main() over the C ABI), linked against libb2blas.so."""
    if _stale(DRIVER_BIN, [DRIVER_SRC, LIB, os.path.join(PKG, "..", "include", "b2blas.h")]):
        cmd = [nvcc(), "-O2", "-std=c++17", "-I" + os.path.join(PKG, "..", "include"), DRIVER_SRC, "-o", DRIVER_BIN,
               "-L" + PKG, "-lb2blas", "-cudart", "shared", "-Xlinker", "-rpath," + PKG, "-Xlinker", "-rpath,/usr/local/cuda/lib64"]
        r = subprocess.run(cmd, capture_output=True, text=True)
        if r.returncode != 0:
            raise RuntimeError("driver build failed:\n" + " ".join(cmd) + "\n" + r.stdout + r.stderr)
    return DRIVER_BIN


CALLS_SRC = os.path.join(CSRC, "calls.cpp")
CALLS = os.path.join(PKG, "_calls.so")
CALLS_STAMP = os.path.join(OBJ, "calls.stamp")


def _torch() -> tuple[str, str] | None:
    """(folder, version) of the torch that the extension can be built against, found without importing it; None without a torch for
    CUDA: the library and the driver need none."""
    spec = importlib.util.find_spec("torch")
    at = spec.submodule_search_locations[0] if spec and spec.submodule_search_locations else None
    if at is None or not glob.glob(os.path.join(at, "lib", "libc10_cuda.so*")):
        return None
    with open(os.path.join(at, "version.py")) as f:
        found = re.search(r"__version__\s*=\s*['\"]([^'\"]+)", f.read())
    return (at, found.group(1)) if found else None


def build_calls(force: bool = False) -> str | None:
    """The extension module ``_calls``, against the torch it will run with: made again when that is another one than last time.
    Without a torch for CUDA, or without Python's headers, there is none (None is returned), and ``layer.py`` makes every call itself."""
    found = _torch()
    if found is None or not os.path.exists(os.path.join(sysconfig.get_paths()["include"], "Python.h")):
        sys.stderr.write("no torch for CUDA, or no Python.h: the extension of layer.py's calls is not built\n")
        return None
    at, version = found
    stamp = f"{version} {sys.implementation.cache_tag} {at}"
    try:
        with open(CALLS_STAMP) as f:
            same = f.read() == stamp
    except OSError:
        same = False
    if force or not same or _stale(CALLS, [CALLS_SRC, os.path.join(PKG, "..", "include", "b2blas.h")]):
        import torch
        cuda = os.path.dirname(os.path.dirname(nvcc()))
        cmd = ["g++", "-O2", "-std=c++17", "-fPIC", "-shared", "-I" + sysconfig.get_paths()["include"], "-I" + os.path.join(at, "include"),
               "-I" + os.path.join(at, "include", "torch", "csrc", "api", "include"), "-I" + os.path.join(cuda, "include"), CALLS_SRC, "-o", CALLS,
               f'-DB2_BUILT_FOR_TORCH="{version}"', "-D_GLIBCXX_USE_CXX11_ABI=%d" % torch._C._GLIBCXX_USE_CXX11_ABI, "-L" + os.path.join(at, "lib"),
               "-Wl,-rpath," + os.path.join(at, "lib"), "-ltorch_python", "-ltorch", "-ltorch_cpu", "-lc10_cuda", "-lc10"]
        r = subprocess.run(cmd, capture_output=True, text=True)
        if r.returncode != 0:
            raise RuntimeError("extension build failed:\n" + " ".join(cmd) + "\n" + r.stdout + r.stderr)
        with open(CALLS_STAMP, "w") as f:
            f.write(stamp)
    return CALLS


if __name__ == "__main__":
    path = build(verbose=True, force="--force" in sys.argv, ptxas_info="--ptxas" in sys.argv)
    print(path)
