"""Build the sm_100a decode library in-tree.

    python mamba3-fused-triton-kernel_b200/build_native.py [--ptxas-verbose] [--force]

Compiles every ``csrc/*.cu`` with nvcc for ``sm_100a`` (one process per file,
in parallel) and links ``lib/libmamba3_b200.so`` with the CUDA runtime linked
statically, so the library only needs the driver at run time.  Objects go to
``_build/`` next to this file.  A file is rebuilt when it or any header under
``csrc/`` / the repository ``include/`` is newer than its object.  Also builds
``lib/m3_host.so`` from ``csrc/m3_host.cpp`` (a Python module on PyTorch's C++
interface, no CUDA code): the host-side fast path of the language-model
operators, left out where PyTorch or g++ is missing.
"""

from __future__ import annotations

import argparse
import concurrent.futures as cf
import glob
import os
import shutil
import subprocess
import sys
import sysconfig

HERE = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(HERE)
CSRC = os.path.join(HERE, "csrc")
INCLUDE = os.path.join(ROOT, "include")
BUILD = os.path.join(HERE, "_build")
LIBDIR = os.path.join(HERE, "lib")
LIB = os.path.join(LIBDIR, "libmamba3_b200.so")
HOST_SRC = os.path.join(CSRC, "m3_host.cpp")
HOST_LIB = os.path.join(LIBDIR, "m3_host.so")
HOST_STAMP = os.path.join(BUILD, "m3_host.torch")  # the PyTorch it was built with

ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]
CFLAGS = ["-O3", "-std=c++17", "-lineinfo", "-Xcompiler", "-fPIC,-O3",
          "--expt-relaxed-constexpr", "-I" + INCLUDE, "-I" + CSRC]


def _nvcc() -> str:
    for cand in (os.environ.get("NVCC"), shutil.which("nvcc"), "/usr/local/cuda/bin/nvcc"):
        if cand and os.path.exists(cand):
            return cand
    raise RuntimeError("nvcc not found (set NVCC or put /usr/local/cuda/bin on PATH)")


def _headers_mtime() -> float:
    hs = glob.glob(os.path.join(CSRC, "*.cuh")) + glob.glob(os.path.join(INCLUDE, "*.h"))
    return max((os.path.getmtime(h) for h in hs), default=0.0)


def _compile(nvcc: str, src: str, obj: str, ptxas_verbose: bool) -> str:
    cmd = [nvcc, *ARCH, *CFLAGS, "-c", src, "-o", obj]
    if ptxas_verbose:
        cmd.insert(1, "-Xptxas=-v")
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"nvcc failed on {os.path.basename(src)}:\n{r.stdout}\n{r.stderr}")
    return r.stderr if ptxas_verbose else ""


def build(force: bool = False, ptxas_verbose: bool = False, jobs: int = 0) -> str:
    """Compile and link; returns the path of the shared library."""
    nvcc = _nvcc()
    os.makedirs(BUILD, exist_ok=True)
    os.makedirs(LIBDIR, exist_ok=True)
    hdr = _headers_mtime()
    srcs = sorted(glob.glob(os.path.join(CSRC, "*.cu")))
    todo, objs = [], []
    for s in srcs:
        o = os.path.join(BUILD, os.path.basename(s)[:-3] + ".o")
        objs.append(o)
        if force or ptxas_verbose or not os.path.exists(o) or os.path.getmtime(o) < max(os.path.getmtime(s), hdr):
            todo.append((s, o))
    logs = []
    if todo:
        n = jobs or min(len(todo), os.cpu_count() or 4)
        with cf.ThreadPoolExecutor(max_workers=n) as ex:
            futs = [ex.submit(_compile, nvcc, s, o, ptxas_verbose) for s, o in todo]
            for f in futs:
                logs.append(f.result())
    if todo or not os.path.exists(LIB) or os.path.getmtime(LIB) < max(os.path.getmtime(o) for o in objs):
        tmp = LIB + ".tmp"
        cmd = [nvcc, *ARCH, "-shared", "-Xcompiler", "-fPIC", "-o", tmp, *objs]
        r = subprocess.run(cmd, capture_output=True, text=True)
        if r.returncode != 0:
            raise RuntimeError(f"link failed:\n{r.stdout}\n{r.stderr}")
        os.replace(tmp, LIB)
    if ptxas_verbose:
        sys.stderr.write("".join(logs))
    build_host(nvcc, force)
    return LIB


def build_host(nvcc: str, force: bool = False) -> bool:
    """``lib/m3_host.so``, with the C++ compiler and the headers of the
    PyTorch that this interpreter imports; rebuilt for another PyTorch, whose
    objects may be laid out differently.  Where one of them is missing it is
    left out with a warning: the operators then take the Python path.  True
    if the module stands."""
    try:
        import torch
        base, version = os.path.dirname(torch.__file__), str(torch.__version__)
    except ImportError:
        base = version = None
    newest = max(os.path.getmtime(HOST_SRC), *(os.path.getmtime(h) for h in glob.glob(os.path.join(INCLUDE, "*.h"))))
    if not force and os.path.exists(HOST_LIB) and os.path.getmtime(HOST_LIB) >= newest and \
            version is not None and _host_version() == version:
        return True
    cxx = shutil.which("g++")
    missing = "PyTorch" if base is None else "g++" if cxx is None else \
        None if os.path.exists(os.path.join(base, "include", "torch", "csrc", "Exceptions.h")) else "PyTorch's headers"
    if missing is not None:
        if os.path.exists(HOST_LIB):
            os.remove(HOST_LIB)  # of other sources than the library, or for another PyTorch
        print(f"warning: {missing} not found, {os.path.basename(HOST_LIB)} is left out", file=sys.stderr)
        return False

    inc = [os.path.join(base, "include"), os.path.join(base, "include", "torch", "csrc", "api", "include"),
           sysconfig.get_paths()["include"], os.path.join(os.path.dirname(os.path.dirname(nvcc)), "include"), INCLUDE]
    libs = os.path.join(base, "lib")
    tmp = HOST_LIB + ".tmp"
    cmd = [cxx, "-O2", "-std=c++17", "-fPIC", "-shared", "-fvisibility=hidden",
           f'-DM3_TORCH_VERSION="{version}"', f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
           *("-I" + i for i in inc), HOST_SRC, "-o", tmp, "-L" + libs, "-ltorch_python", "-ltorch", "-ltorch_cpu", "-lc10", "-lc10_cuda"]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"g++ failed on {os.path.basename(HOST_SRC)}:\n{r.stdout}\n{r.stderr}")
    os.replace(tmp, HOST_LIB)
    with open(HOST_STAMP, "w") as f:
        f.write(version)
    return True


def _host_version() -> str | None:
    """The PyTorch that the module was built with."""
    try:
        with open(HOST_STAMP) as f:
            return f.read()
    except OSError:
        return None


def main():
    ap = argparse.ArgumentParser()
    ap.add_argument("--force", action="store_true")
    ap.add_argument("--ptxas-verbose", action="store_true")
    ap.add_argument("--jobs", type=int, default=0)
    a = ap.parse_args()
    print(build(force=a.force, ptxas_verbose=a.ptxas_verbose, jobs=a.jobs))


if __name__ == "__main__":
    main()
