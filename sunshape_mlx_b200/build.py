"""Builds libsunshape_b200.so (all CUDA sources, sm_100a) and, where torch is
installed, the native lane of the paged wrappers (_fast, a CPython extension
over it) in place.

    python -m sunshape_mlx_b200.build          # or: python sunshape_mlx_b200/build.py

nvcc cross-compiles for sm_100a without a GPU. An object is rebuilt only when
its source or a header is newer than it; stale objects compile in parallel.
"""

from __future__ import annotations

import glob
import importlib.util
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
    return ([x for p in inc for x in ("-isystem", p)] + [f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}"],
            ["-L" + os.path.join(root, "lib"), *[f"-l{x}" for x in libs]])


def _have_torch() -> bool:
    return "torch" in sys.modules or importlib.util.find_spec("torch") is not None


def _fresh(target: str, deps: list[str]) -> bool:
    return os.path.exists(target) and all(os.path.getmtime(d) <= os.path.getmtime(target) for d in deps)


def _run(cmds: list[list[str]], verbose: bool) -> None:
    """Runs the commands side by side."""
    procs = []
    for cmd in cmds:
        if verbose:
            print(" ".join(cmd), flush=True)
        procs.append(subprocess.Popen(cmd))
    failed = [c for c, pr in zip(cmds, procs) if pr.wait() != 0]
    if failed:
        raise subprocess.CalledProcessError(1, failed[0])


def build(force: bool = False, verbose: bool = False) -> str:
    """Builds what is out of date: the library, then, where torch is installed, the
    extension over it. The library needs nvcc alone."""
    headers = glob.glob(os.path.join(CSRC, "*.cuh")) + glob.glob(os.path.join(INCLUDE, "*.h"))
    objdir = os.path.join(HERE, "_build")
    if force or not _fresh(LIB, [*sources(), *headers]):
        nvcc = _nvcc()
        os.makedirs(objdir, exist_ok=True)
        objs, cmds = [], []
        for src in sources():
            obj = os.path.join(objdir, os.path.basename(src)[:-3] + ".o")
            objs.append(obj)
            if force or not _fresh(obj, [src, *headers]):
                cmds.append([nvcc, *ARCH, *FLAGS, "-I", INCLUDE, "-c", src, "-o", obj])
        _run(cmds, verbose)
        _run([[nvcc, *ARCH, "-shared", "-o", LIB + ".tmp", *objs, "-lcudart"]], verbose)
        os.replace(LIB + ".tmp", LIB)
    if _have_torch() and (force or not _fresh(FAST, [FAST_SRC, *glob.glob(os.path.join(INCLUDE, "*.h"))])):
        os.makedirs(objdir, exist_ok=True)
        inc, link = _torch_flags()
        obj = os.path.join(objdir, "binding.o")
        _run([["g++", "-O2", "-std=c++17", "-fPIC", "-Wall", *inc, "-c", FAST_SRC, "-o", obj]], verbose)
        _run([["g++", "-shared", "-o", FAST + ".tmp", obj, "-L" + HERE, "-lsunshape_b200", *link, "-Wl,-rpath,$ORIGIN"]], verbose)
        os.replace(FAST + ".tmp", FAST)
    return LIB


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose=True))
