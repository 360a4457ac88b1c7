"""Builds libsunshape_b200.so (all CUDA sources, sm_100a) and the native lane
of the paged wrappers (_fast, a CPython extension over it) in place.

    python -m sunshape_mlx_b200.build          # or: python sunshape_mlx_b200/build.py

nvcc cross-compiles for sm_100a without a GPU. An object is rebuilt only when
its source or a header is newer than it; stale objects compile in parallel.
"""

from __future__ import annotations

import glob
import os
import shutil
import subprocess
import sys
import sysconfig

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
INCLUDE = os.path.join(os.path.dirname(HERE), "include")
LIB = os.path.join(HERE, "libsunshape_b200.so")
FAST_SRC = os.path.join(CSRC, "binding.cpp")
FAST = os.path.join(HERE, "_fast" + (sysconfig.get_config_var("EXT_SUFFIX") or ".so"))
ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]
FLAGS = ["-O3", "-std=c++17", "-lineinfo", "-Xcompiler", "-fPIC", "--expt-relaxed-constexpr",
         "-Xcompiler", "-Wall", "-Xcompiler", "-Wno-unused-function"]


def _nvcc() -> str:
    for cand in (shutil.which("nvcc"), "/usr/local/cuda/bin/nvcc"):
        if cand and os.path.exists(cand):
            return cand
    raise RuntimeError("nvcc not found: the SunShape CUDA library cannot be built")


def sources() -> list[str]:
    return sorted(glob.glob(os.path.join(CSRC, "*.cu")))


def _torch_flags() -> tuple[list[str], list[str]]:
    """(include, link) flags of the extension; torch's own folders, no CUDA probing."""
    import torch

    root = os.path.dirname(torch.__file__)
    inc = [os.path.join(root, "include"), os.path.join(root, "include", "torch", "csrc", "api", "include"),
           sysconfig.get_paths()["include"], os.path.join(os.path.dirname(os.path.dirname(_nvcc())), "include")]
    libs = ["torch_python", "torch", "torch_cpu", "c10", "c10_cuda"]
    return ([f"-I{p}" for p in inc] + [f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}"],
            ["-L" + os.path.join(root, "lib"), *[f"-l{x}" for x in libs]])


def _stale() -> bool:
    if not os.path.exists(LIB) or not os.path.exists(FAST):
        return True
    t = min(os.path.getmtime(LIB), os.path.getmtime(FAST))
    deps = sources() + [FAST_SRC] + glob.glob(os.path.join(CSRC, "*.cuh")) + glob.glob(os.path.join(INCLUDE, "*.h"))
    return any(os.path.getmtime(f) > t for f in deps)


def build(force: bool = False, verbose: bool = False) -> str:
    if not force and not _stale():
        return LIB
    nvcc = _nvcc()
    objdir = os.path.join(HERE, "_build")
    os.makedirs(objdir, exist_ok=True)
    headers = glob.glob(os.path.join(CSRC, "*.cuh")) + glob.glob(os.path.join(INCLUDE, "*.h"))
    objs, cmds = [], []
    for src in sources():
        obj = os.path.join(objdir, os.path.basename(src)[:-3] + ".o")
        objs.append(obj)
        fresh = os.path.exists(obj) and all(
            os.path.getmtime(d) <= os.path.getmtime(obj) for d in [src, *headers])
        if force or not fresh:
            cmds.append([nvcc, *ARCH, *FLAGS, "-I", INCLUDE, "-c", src, "-o", obj])
    inc, link = _torch_flags()
    fast_obj = os.path.join(objdir, "binding.o")
    if force or not (os.path.exists(fast_obj) and all(
            os.path.getmtime(d) <= os.path.getmtime(fast_obj) for d in [FAST_SRC, *glob.glob(os.path.join(INCLUDE, "*.h"))])):
        cmds.append(["g++", "-O2", "-std=c++17", "-fPIC", "-w", *inc, "-c", FAST_SRC, "-o", fast_obj])
    # objects compile independently: run them side by side
    procs = []
    for cmd in cmds:
        if verbose:
            print(" ".join(cmd), flush=True)
        procs.append(subprocess.Popen(cmd))
    failed = [c for c, pr in zip(cmds, procs) if pr.wait() != 0]
    if failed:
        raise subprocess.CalledProcessError(1, failed[0])
    tmp = LIB + ".tmp"
    cmd = [nvcc, *ARCH, "-shared", "-o", tmp, *objs, "-lcudart"]
    if verbose:
        print(" ".join(cmd), flush=True)
    subprocess.run(cmd, check=True)
    os.replace(tmp, LIB)
    cmd = ["g++", "-shared", "-o", FAST + ".tmp", fast_obj, "-L" + HERE, "-lsunshape_b200", *link, "-Wl,-rpath,$ORIGIN"]
    if verbose:
        print(" ".join(cmd), flush=True)
    subprocess.run(cmd, check=True)
    os.replace(FAST + ".tmp", FAST)
    return LIB


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose=True))
