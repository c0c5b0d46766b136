"""Builds libaf2cuda.so in-tree with nvcc for sm_100a.

    python alphafold2-webgpu_b200/build.py [--verbose]

Each .cu under csrc/ is compiled to an object (in csrc/_build/, git-ignored)
with `-gencode arch=compute_100a,code=sm_100a -lineinfo -O3`, then linked
into alphafold2-webgpu_b200/libaf2cuda.so with the CUDA runtime linked
statically, so the library needs only the driver at run time.

The package's torch glue, af2cuda/_tensors.cpp, is compiled with g++ against
the headers of the installed torch into af2cuda/_tensors.so; only the learned
layers' entry points on torch tensors use it.
"""
from __future__ import annotations

import os
import shutil
import subprocess
import sys
from concurrent.futures import ThreadPoolExecutor
from pathlib import Path

PKG = Path(__file__).resolve().parent
CSRC = PKG / "csrc"
BUILD = CSRC / "_build"
LIB = PKG / "libaf2cuda.so"
INCLUDE = PKG.parent / "include"

ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]
FLAGS = ["-O3", "-lineinfo", "-std=c++17", "-Xcompiler", "-fPIC,-fvisibility=hidden", "--expt-relaxed-constexpr",
         "-I", str(INCLUDE)]


def nvcc() -> str:
    cand = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    if not Path(cand).exists():
        raise RuntimeError("nvcc not found; the CUDA 12.9 toolkit is required to build libaf2cuda.so")
    return cand


def _compile(src: Path, verbose: bool) -> Path:
    obj = BUILD / (src.stem + ".o")
    deps = [src] + list(CSRC.glob("*.cuh")) + list(CSRC.glob("*.h")) + list(INCLUDE.glob("*.h"))
    if obj.exists() and obj.stat().st_mtime >= max(d.stat().st_mtime for d in deps):
        return obj
    cmd = [nvcc(), *ARCH, *FLAGS, "-c", str(src), "-o", str(obj)]
    if verbose:
        cmd.insert(1, "-Xptxas=-v")
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError(f"nvcc failed on {src.name}:\n{res.stderr}")
    if verbose:
        sys.stderr.write(res.stderr)
    return obj


def build_tensors() -> Path:
    """af2cuda/_tensors.so, against this interpreter's torch."""
    import sysconfig

    import torch
    src, out = PKG / "af2cuda" / "_tensors.cpp", PKG / "af2cuda" / "_tensors.so"
    stamp = BUILD / "_tensors.torch"  # the torch it was built against
    deps = [src] + list(INCLUDE.glob("*.h"))
    if out.exists() and stamp.exists() and stamp.read_text() == torch.__version__ \
            and out.stat().st_mtime >= max(d.stat().st_mtime for d in deps):
        return out
    from torch.utils.cpp_extension import include_paths, library_paths
    cuda = Path(nvcc()).resolve().parent.parent
    cmd = [shutil.which("g++") or "g++", "-O2", "-std=c++17", "-shared", "-fPIC", "-fvisibility=hidden",
           f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
           *(a for p in [*include_paths(), sysconfig.get_paths()["include"], str(cuda / "include")]
             for a in ("-isystem", p)), "-I", str(INCLUDE), str(src), "-o", str(out),
           *(f"-L{p}" for p in library_paths()), "-lc10", "-lc10_cuda", "-ltorch_cpu", "-ltorch_python"]
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError(f"g++ failed on {src.name}:\n{res.stderr}")
    stamp.write_text(torch.__version__)
    return out


def build(verbose: bool = False) -> Path:
    BUILD.mkdir(exist_ok=True)
    build_tensors()
    sources = sorted(CSRC.glob("*.cu"))
    with ThreadPoolExecutor(max_workers=min(8, os.cpu_count() or 1)) as pool:
        objs = list(pool.map(lambda s: _compile(s, verbose), sources))
    if LIB.exists() and LIB.stat().st_mtime >= max(o.stat().st_mtime for o in objs):
        return LIB
    # NCCL is not linked: the library opens the process's libnccl.so.2 when a
    # communicator is first created (comm.cu), so it never brings a second copy.
    cmd = [nvcc(), *ARCH, "-shared", "-o", str(LIB), *map(str, objs), "-cudart", "static", "-ldl"]
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError(f"link failed:\n{res.stderr}")
    return LIB


if __name__ == "__main__":
    print(build(verbose="--verbose" in sys.argv))
