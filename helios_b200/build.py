"""Builds libg4q.so (the C-ABI kernel library) in-tree with nvcc for sm_100a, and, where torch can be imported,
_g4q_torch (the Python side of the attention calls, a CPython module over torch's headers) with the host compiler.

``python -m helios_b200.build`` or ``helios_b200.build.build()``. The shared library lands
next to this file so it travels with the source tree; no JIT cache is involved.
"""
from __future__ import annotations

import os
import subprocess
import sys
from pathlib import Path

from . import _lib

PKG = Path(__file__).resolve().parent
ROOT = PKG.parent
CSRC = PKG / "csrc"
INCLUDE = ROOT / "include"
LIB = PKG / "libg4q.so"
TORCH_SRC = CSRC / "g4q_torch.cpp"
OBJDIR = PKG / "_build"

SOURCES = ["g4q_api.cu", "g4q_layout.cu", "g4q_gemv.cu", "g4q_gemv2.cu", "g4q_gemm.cu", "g4q_decode.cu",
           "g4q_generic.cu", "g4q_comm.cu", "g4q_lora.cu", "g4q_mlp.cu", "g4q_rope.cu",
           "g4q_attn.cu", "g4q_attn_chunk.cu"]
HEADERS = ["g4q_common.cuh", "g4q_internal.h", "g4q_overlap.h", "g4q_attn.cuh"]

NVCC_FLAGS = [
    "-gencode", "arch=compute_100a,code=sm_100a",
    "-O3", "-lineinfo", "-std=c++17",
    "-Xcompiler", "-fPIC,-O3",
    "--expt-relaxed-constexpr",
    "-Xptxas", "-warn-spills",
]


def _nvcc() -> str:
    cand = os.environ.get("NVCC") or "/usr/local/cuda/bin/nvcc"
    return cand if Path(cand).exists() else "nvcc"


def _stale(target: Path, deps) -> bool:
    if not target.exists():
        return True
    t = target.stat().st_mtime
    return any(Path(d).stat().st_mtime > t for d in deps)


def _torch_command(torch, target: Path) -> list:
    """The host compiler's command for _g4q_torch."""
    import sysconfig

    root = Path(torch.__file__).resolve().parent
    inc = [root / "include", root / "include" / "torch" / "csrc" / "api" / "include", sysconfig.get_paths()["include"],
           INCLUDE]
    return [os.environ.get("CXX", "g++"), "-O2", "-std=c++17", "-fPIC", "-shared",
            f"-D_GLIBCXX_USE_CXX11_ABI={int(torch.compiled_with_cxx11_abi())}", *(f"-I{i}" for i in inc), str(TORCH_SRC),
            "-o", str(target), f"-L{root / 'lib'}", "-ltorch_python", "-ltorch_cpu", "-lc10"]


def build(verbose: bool = False, force: bool = False) -> Path:
    """Compile every .cu under csrc/ for sm_100a and link libg4q.so, whose path is returned; build _g4q_torch beside it
    where torch can be imported (the C ABI needs none of it)."""
    OBJDIR.mkdir(exist_ok=True)
    nvcc = _nvcc()
    common_deps = [CSRC / h for h in HEADERS] + [INCLUDE / "g4q.h"]
    objs, cmds = [], []
    for src in SOURCES:
        obj = OBJDIR / (src + ".o")
        objs.append(obj)
        if force or _stale(obj, [CSRC / src] + common_deps):
            cmds.append([nvcc, *NVCC_FLAGS, "-I", str(INCLUDE), "-I", str(CSRC), "-c", str(CSRC / src), "-o", str(obj)])
    module_cmd = None
    try:
        import torch
        target = _lib.torch_module_path(torch.__version__)
        if force or _stale(target, [TORCH_SRC, INCLUDE / "g4q.h"]):
            module_cmd = _torch_command(torch, target)
    except ImportError as e:
        print(f"_g4q_torch is not built, torch cannot be imported: {e}", file=sys.stderr, flush=True)
    # translation units compile independently: one nvcc per source, a few at a time
    from concurrent.futures import ThreadPoolExecutor

    def compile_one(cmd):
        if verbose:
            print(" ".join(cmd), flush=True)
        subprocess.run(cmd, check=True)

    with ThreadPoolExecutor(max_workers=min(8, os.cpu_count() or 1)) as ex:
        module = ex.submit(compile_one, module_cmd) if module_cmd else None
        list(ex.map(compile_one, cmds))
        if force or _stale(LIB, objs):
            compile_one([nvcc, "-gencode", "arch=compute_100a,code=sm_100a", "-shared", "-o", str(LIB), *map(str, objs),
                         "-lcudart", "-Xlinker", "-z,defs"])
        if module is not None:
            module.result()      # the library is complete, whatever became of the module
    return LIB


if __name__ == "__main__":
    build(verbose=True, force="--force" in sys.argv)
