"""Builds libcafe_b200.so in-tree with nvcc for sm_100a, and _dense_torch.so with g++.

    python -m cafe_b200.build [--force]

The library is a plain C-ABI shared object (include/cafe_b200.h) that does not link against torch.  _dense_torch.so, the
autograd nodes of the dense layers and AdamW's calls, links against it and torch.
"""
from __future__ import annotations

import os
import subprocess
import sys
from pathlib import Path

PKG = Path(__file__).resolve().parent
CSRC = PKG / "csrc"
SO = PKG / "libcafe_b200.so"
SOURCES = ["sketch_cuda.cu", "embed_cuda.cu", "sigmod_cuda.cu", "interact_cuda.cu", "dense_cuda.cu", "dense_tiles.cu", "adamw_cuda.cu", "ref_abi.cu", "prof.cu"]
HEADERS = ["cafe_types.h", "cafe_internal.h", "sketch_core.cuh", "sketch_engine.h", "radix_sort.cuh", "cafe_float.cuh", "tcgen05.cuh", "dense.cuh"]
TORCH_SO = PKG / "_dense_torch.so"
TORCH_SOURCE = CSRC / "dense_torch.cpp"
TORCH_RECORD = PKG / "build" / "_dense_torch.built_for"   # what TORCH_SO was built for: it loads with no other torch or python
NVCC_FLAGS = ["-gencode", "arch=compute_100a,code=sm_100a", "-lineinfo", "-O3", "-std=c++17", "-Xcompiler", "-fPIC",
              "--expt-relaxed-constexpr"]
# the sketch arithmetic must not be contracted into fused multiply-adds: counts are compared bit for bit
PER_FILE = {"sketch_cuda.cu": ["-fmad=false"], "sigmod_cuda.cu": ["-fmad=false"], "ref_abi.cu": ["-fmad=false"], "embed_cuda.cu": [],
            "prof.cu": [], "interact_cuda.cu": [], "dense_cuda.cu": [], "dense_tiles.cu": [], "adamw_cuda.cu": []}


def _nvcc() -> str:
    for c in (os.environ.get("NVCC"), "/usr/local/cuda/bin/nvcc", "nvcc"):
        if c and (Path(c).exists() or c == "nvcc"):
            return c
    raise RuntimeError("nvcc not found")


def _stale() -> bool:
    if not SO.exists():
        return True
    t = SO.stat().st_mtime
    deps = [CSRC / s for s in SOURCES + HEADERS] + [PKG.parent / "include" / "cafe_b200.h", Path(__file__)]
    return any(d.stat().st_mtime > t for d in deps)


def build(force: bool = False, verbose: bool = False) -> Path:
    if not force and not _stale():
        return SO
    nvcc = _nvcc()
    objdir = PKG / "build"
    objdir.mkdir(exist_ok=True)
    procs = []
    for s in SOURCES:
        obj = objdir / (s + ".o")
        cmd = [nvcc, *NVCC_FLAGS, *PER_FILE[s], "-c", str(CSRC / s), "-o", str(obj)]
        if verbose:
            cmd.insert(1, "-Xptxas")
            cmd.insert(2, "-v")
        procs.append((s, obj, subprocess.Popen(cmd, stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True)))
    objs = []
    for s, obj, p in procs:
        out, _ = p.communicate()
        if p.returncode != 0:
            raise RuntimeError(f"nvcc failed on {s}:\n{out}")
        if verbose:
            print(out)
        objs.append(str(obj))
    link = [nvcc, "-shared", "-o", str(SO), *objs, "-lcudart"]
    r = subprocess.run(link, stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"link failed:\n{r.stdout}")
    return SO


def build_torch(force: bool = False) -> Path:
    """The extension module cafe_b200._dense_torch (after build(): it is linked against the library)."""
    from importlib.metadata import version
    built_for = f"torch {version('torch')}, python {sys.version}"
    deps = [TORCH_SOURCE, PKG.parent / "include" / "cafe_b200.h", Path(__file__)]
    if not force and TORCH_SO.exists() and all(d.stat().st_mtime <= TORCH_SO.stat().st_mtime for d in deps) and \
            TORCH_RECORD.exists() and TORCH_RECORD.read_text() == built_for:
        return TORCH_SO
    import sysconfig

    import torch
    from torch.utils import cpp_extension
    nvcc = Path(_nvcc())
    cuda = [f"-I{nvcc.parent.parent / 'include'}"] if nvcc.is_absolute() else []
    # (g++ itself, whatever CXX says: a second libstdc++ linked into the module would crash on the first formatted message)
    cmd = ["g++", "-O2", "-std=c++17", "-fPIC", "-shared", f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
           *[f"-I{p}" for p in cpp_extension.include_paths()], *cuda, f"-I{sysconfig.get_paths()['include']}", str(TORCH_SOURCE), "-o", str(TORCH_SO),
           *[f"-L{p}" for p in cpp_extension.library_paths()], f"-L{PKG}", "-Wl,-rpath,$ORIGIN", f"-l:{SO.name}", "-lc10", "-lc10_cuda", "-ltorch_cpu",
           "-ltorch", "-ltorch_python"]
    r = subprocess.run(cmd, stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"g++ failed on {TORCH_SOURCE.name}:\n{r.stdout}")
    TORCH_RECORD.parent.mkdir(exist_ok=True)
    TORCH_RECORD.write_text(built_for)
    return TORCH_SO


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose="-v" in sys.argv))
    print(build_torch(force="--force" in sys.argv))
