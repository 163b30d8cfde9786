"""Build recipe of libade_b200.so (the CUDA kernels behind the C ABI of include/ade_b200.h).

`python -m ade_b200.build` compiles the .cu files of ade_b200/csrc for sm_100a with nvcc, side by side, and puts
the shared object next to this file, where ade_b200._lib loads it.  nvcc cross-compiles, so
the build needs no GPU.  The explicit -gencode form is required: tcgen05 instructions only
exist for the architecture-specific target sm_100a.
"""
from __future__ import annotations

import os
import subprocess
import sys

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
LIB = os.path.join(HERE, "libade_b200.so")
SHIM = os.path.join(HERE, "libade_b200_torch.so")
NVCC_FLAGS = [
    "-gencode", "arch=compute_100a,code=sm_100a", "-O3", "-lineinfo", "-std=c++17",
    "-Xcompiler", "-fPIC",
]
SHIM_SOURCES = ("torch_shim.cpp", "torch_requests.cpp")


def sources():
    return [os.path.join(CSRC, f) for f in sorted(os.listdir(CSRC)) if f.endswith((".cu", ".cuh", ".h"))] + [
        os.path.join(os.path.dirname(HERE), "include", "ade_b200.h")]


def _current(obj: str, src: str) -> bool:
    """Whether the object file is newer than its source, the headers that the source includes, directly or not, and this recipe."""
    if not os.path.exists(obj):
        return False
    seen, todo = set(), [src, os.path.abspath(__file__)]
    while todo:
        f = todo.pop()
        if f in seen or not os.path.exists(f):
            continue
        seen.add(f)
        if f.endswith(".py"):
            continue
        with open(f) as text:
            todo += [os.path.normpath(os.path.join(os.path.dirname(f), line.split('"')[1])) for line in text if line.startswith('#include "')]
    return all(os.path.getmtime(obj) >= os.path.getmtime(f) for f in seen)


def build(force: bool = False, verbose: bool = False) -> str:
    """Compile the kernel library and the torch binding when they are missing or older than any of their sources."""
    if force or not (os.path.exists(LIB) and all(os.path.getmtime(LIB) >= os.path.getmtime(s) for s in sources())):
        nvcc = os.path.join(os.environ.get("CUDA_HOME", "/usr/local/cuda"), "bin", "nvcc")
        flags = [*NVCC_FLAGS, *(["-Xptxas", "-v"] if verbose else [])]
        units = {s: s[:-3] + ".o" for s in sources() if s.endswith(".cu")}
        stale = [s for s, o in units.items() if force or not _current(o, s)]
        jobs = [subprocess.Popen([nvcc, *flags, "-c", s, "-o", units[s] + ".tmp"]) for s in stale]
        if any([j.wait() for j in jobs]):
            raise subprocess.CalledProcessError(1, [nvcc, *flags, "-c", *stale])
        for s in stale:
            os.replace(units[s] + ".tmp", units[s])
        subprocess.run([nvcc, *NVCC_FLAGS, "-shared", *units.values(), "-o", LIB + ".tmp"], check=True)
        os.replace(LIB + ".tmp", LIB)
    build_shim(force)
    return LIB


def build_shim(force: bool = False) -> str:
    """The thin torch binding (csrc/torch_*.cpp -> libade_b200_torch.so): host compiler only, linked against the
    kernel library next to it (found at run time through $ORIGIN) and against the installed torch."""
    srcs = [os.path.join(CSRC, f) for f in SHIM_SOURCES]
    header = os.path.join(os.path.dirname(HERE), "include", "ade_b200.h")
    if not force and os.path.exists(SHIM) and all(os.path.getmtime(SHIM) >= os.path.getmtime(s) for s in (*srcs, header, LIB)):
        return SHIM
    import torch
    from torch.utils import cpp_extension as ce

    inc = ce.include_paths("cuda")
    libs = ce.library_paths("cuda")
    abi = int(torch._C._GLIBCXX_USE_CXX11_ABI)
    flags = ["-O2", "-std=c++17", "-fPIC", f"-D_GLIBCXX_USE_CXX11_ABI={abi}", *[f"-I{i}" for i in inc]]
    objs = [s[:-4] + ".o" for s in srcs]
    jobs = [subprocess.Popen(["g++", *flags, "-c", s, "-o", o]) for s, o in zip(srcs, objs)]
    if any([j.wait() for j in jobs]):
        raise subprocess.CalledProcessError(1, ["g++", *flags, "-c", *srcs])
    cmd = ["g++", "-shared", *objs, "-o", SHIM + ".tmp", *[f"-L{l}" for l in libs], f"-L{HERE}", "-lade_b200", "-lc10", "-lc10_cuda", "-ltorch_cpu",
           "-ltorch_cuda", "-ltorch", "-Wl,-rpath,$ORIGIN", *[f"-Wl,-rpath,{l}" for l in libs]]
    subprocess.run(cmd, check=True)
    os.replace(SHIM + ".tmp", SHIM)
    return SHIM


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose="-v" in sys.argv))
