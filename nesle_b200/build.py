"""Builds libnesle_b200.so in-tree for sm_100a (nvcc; no JIT cache).

    python -m nesle_b200.build          # incremental
    python -m nesle_b200.build --force  # rebuild
"""
from __future__ import annotations

import argparse
import os
import shutil
import subprocess
import sys
from concurrent.futures import ThreadPoolExecutor
from pathlib import Path

PKG = Path(__file__).resolve().parent
CSRC = PKG / "csrc"
ROOT = PKG.parent
LIB = PKG / "libnesle_b200.so"
OBJ = CSRC / "_build"
_CORE = ["kernels.h", "nes_core.cuh", "nes_render.cuh", "nes_v2.cuh", "nesle_state.h", "formats.h"]
_OPS = ["ops_common.h", "tc05.cuh"]
# source -> the headers it includes; each source is one object, compiled when it or a header is newer
SOURCES = {"kernels.cu": _CORE, "capi.cu": _CORE, "formats.cpp": _CORE, "ops_common.cu": _OPS, "ops_int8.cu": _OPS,
           "ops_orth.cu": _OPS,
           **{f"ops_delta{t}.cu": [*_OPS, "ops_delta.cuh"] for t in ("", "_bf16", "_f16", "_f32")}}
HEADERS = [ROOT / "include" / "nesle_b200.h", ROOT / "include" / "nesle_ops.h"]
ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]


def nvcc() -> str:
    exe = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    if not Path(exe).exists():
        raise RuntimeError("nvcc not found: the CUDA toolkit is required to build libnesle_b200.so")
    return exe


def _newest(src: str) -> float:
    return max(p.stat().st_mtime for p in [CSRC / src, *(CSRC / h for h in SOURCES[src]), *HEADERS])


def needs_build() -> bool:
    return not LIB.exists() or any(_newest(s) > LIB.stat().st_mtime for s in SOURCES)


def build(force: bool = False, verbose: bool = False) -> Path:
    if not force and not needs_build():
        return LIB
    OBJ.mkdir(exist_ok=True)
    flags = ["-std=c++20", "-O3", *ARCH, "-lineinfo", "-Xcompiler", "-fPIC", "-I", str(ROOT / "include")]
    if verbose:
        flags.insert(0, "-Xptxas=-v")

    def compile_one(src: str) -> Path:
        obj = OBJ / (src + ".o")
        if force or not obj.exists() or _newest(src) > obj.stat().st_mtime:
            tmp = OBJ / f"{src}.{os.getpid()}.tmp.o"
            cmd = [nvcc(), *flags, "-c", "-o", str(tmp), str(CSRC / src)]
            if verbose:
                print(" ".join(cmd), flush=True)
            subprocess.run(cmd, check=True, cwd=str(CSRC))
            os.replace(tmp, obj)
        return obj

    with ThreadPoolExecutor(len(SOURCES)) as pool:
        objects = list(pool.map(compile_one, SOURCES))
    tmp = LIB.with_suffix(".so.tmp")
    subprocess.run([nvcc(), *ARCH, "-shared", "-o", str(tmp), *map(str, objects)], check=True, cwd=str(CSRC))
    os.replace(tmp, LIB)
    return LIB


def main(argv=None) -> int:
    ap = argparse.ArgumentParser()
    ap.add_argument("--force", action="store_true")
    ap.add_argument("-v", "--verbose", action="store_true")
    args = ap.parse_args(argv)
    print(build(force=args.force, verbose=args.verbose))
    return 0


if __name__ == "__main__":
    sys.exit(main())
