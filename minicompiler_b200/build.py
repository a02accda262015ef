"""Builds the native parts of minicompiler-b200 in-tree.

    python -m minicompiler_b200.build            # library + mcc tool
    python -m minicompiler_b200.build --force    # rebuild everything

Outputs (all git-ignored, all travel with the working tree):
    minicompiler_b200/libminicompiler_b200.so    host C++ + CUDA kernels for sm_100a + both C ABIs
    minicompiler_b200/mcc                        the command-line driver

The CUDA sources are compiled for sm_100a only (`-gencode arch=compute_100a,code=sm_100a`);
nvcc cross-compiles, so no GPU is needed to build. The kernel bodies (*.cuh) are also
embedded as text, because a matmul with a fused epilogue is specialised at run time with
NVRTC from that same text.
"""

from __future__ import annotations

import argparse
import concurrent.futures
import os
import shutil
import subprocess
import sys
from pathlib import Path

PKG = Path(__file__).resolve().parent
ROOT = PKG.parent
CSRC = PKG / "csrc"
OBJ = PKG / "build"
CUDA_HOME = Path(os.environ.get("CUDA_HOME", "/usr/local/cuda"))
LIB = PKG / "libminicompiler_b200.so"
MCC = PKG / "mcc"

HOST_SOURCES = [
    "core/ir.cpp",
    "core/mcg.cpp",
    "core/passes.cpp",
    "core/plan.cpp",
    "backend/eltwise_codegen.cpp",
    "backend/reduce_codegen.cpp",
    "backend/lowering.cpp",
    "backend/partition.cpp",
    "backend/row_slicing.cpp",
    "backend/b200_backend.cpp",
    "device/runtime.cpp",
    "device/nccl_layer.cpp",
    "capi/capi.cpp",
]
CUDA_SOURCES = ["kernels/gemm_launch.cu", "kernels/no_alloc.cu", "kernels/fp4_quantize.cu", "kernels/fp4_gemm.cu", "kernels/moe_layer.cu"]
EMBEDDED = {
    "kSourceEpilogue": "kernels/epilogue.cuh",
    "kSourceAsyncCopy": "kernels/async_copy.cuh",
    "kSourceGemmF32": "kernels/gemm_f32_simt.cuh",
    "kSourceGemmTc": "kernels/gemm_tcgen05.cuh",
    "kSourceGemmTc2": "kernels/gemm_tcgen05_2cta.cuh",
    "kSourceSplitkReduce": "kernels/splitk_reduce.cuh",
}

INCLUDES = ["-I", str(CSRC), "-I", str(ROOT / "include"), "-I", str(CUDA_HOME / "include")]
CXXFLAGS = ["-std=c++17", "-O2", "-fPIC", "-ffp-contract=off", "-fvisibility=hidden", "-Wall", "-Wextra",
            "-Wno-unused-parameter"]
NVCCFLAGS = ["-std=c++17", "-O3", "-lineinfo", "-gencode", "arch=compute_100a,code=sm_100a", "-Xcompiler",
             "-fPIC,-fvisibility=hidden", "--expt-relaxed-constexpr"]


def _run(cmd: list[str]) -> None:
    proc = subprocess.run(cmd, capture_output=True, text=True)
    if proc.returncode != 0:
        raise RuntimeError("command failed: " + " ".join(cmd) + "\n" + proc.stdout + proc.stderr)
    if proc.stderr.strip():
        sys.stderr.write(proc.stderr)


def _newest_input() -> float:
    newest = Path(__file__).stat().st_mtime
    for base in (CSRC, ROOT / "include"):
        for p in base.rglob("*"):
            if p.is_file():
                newest = max(newest, p.stat().st_mtime)
    return newest


def _write_embedded() -> Path:
    """kernels/*.cuh -> one .cpp holding each file as a string constant."""
    out = OBJ / "embedded_sources.cpp"
    parts = ["// Generated by minicompiler_b200/build.py from csrc/kernels/*.cuh.\nnamespace mcd {\n"]
    for symbol, rel in EMBEDDED.items():
        text = (CSRC / rel).read_text()
        assert ')MCSRC"' not in text
        # String literals are capped at 64 KiB by some compilers: split on line boundaries.
        chunks, current = [], ""
        for line in text.splitlines(keepends=True):
            if len(current) + len(line) > 12000:
                chunks.append(current)
                current = ""
            current += line
        chunks.append(current)
        body = "\n".join('R"MCSRC(' + c + ')MCSRC"' for c in chunks)
        parts.append(f"extern const char* const {symbol};\nconst char* const {symbol} =\n{body};\n")
    parts.append("}  // namespace mcd\n")
    text = "".join(parts)
    if not out.exists() or out.read_text() != text:
        out.write_text(text)
    return out


def build_library(force: bool = False, verbose: bool = False) -> Path:
    OBJ.mkdir(exist_ok=True)
    newest = _newest_input()
    embedded = _write_embedded()
    jobs: list[tuple[list[str], Path]] = []
    objects: list[Path] = []

    def want(obj: Path) -> bool:
        return force or not obj.exists() or obj.stat().st_mtime < newest

    for rel in HOST_SOURCES:
        src = CSRC / rel
        if not src.exists():
            continue
        obj = OBJ / (rel.replace("/", "_") + ".o")
        objects.append(obj)
        if want(obj):
            jobs.append((["g++", *CXXFLAGS, *INCLUDES, "-c", str(src), "-o", str(obj)], obj))
    obj = OBJ / "embedded_sources.o"
    objects.append(obj)
    if want(obj) or obj.stat().st_mtime < embedded.stat().st_mtime:
        jobs.append((["g++", *CXXFLAGS, "-c", str(embedded), "-o", str(obj)], obj))
    for rel in CUDA_SOURCES:
        src = CSRC / rel
        if not src.exists():
            continue
        obj = OBJ / (rel.replace("/", "_") + ".o")
        objects.append(obj)
        if want(obj):
            jobs.append(([str(CUDA_HOME / "bin" / "nvcc"), *NVCCFLAGS, *INCLUDES, "-c", str(src), "-o", str(obj)], obj))

    if jobs:
        with concurrent.futures.ThreadPoolExecutor(max_workers=min(8, len(jobs))) as pool:
            for fut in [pool.submit(_run, cmd) for cmd, _ in jobs]:
                fut.result()
        if verbose:
            print(f"compiled {len(jobs)} translation unit(s)")
    if jobs or not LIB.exists():
        _run(["g++", "-shared", "-o", str(LIB), *map(str, objects), "-L", str(CUDA_HOME / "lib64"), "-lcudart_static",
              "-ldl", "-lrt", "-lpthread", "-Wl,--no-undefined"])
    return LIB


def build_mcc(force: bool = False) -> Path:
    src = CSRC / "tools" / "mcc.cpp"
    if not src.exists():
        return MCC
    if force or not MCC.exists() or MCC.stat().st_mtime < max(_newest_input(), LIB.stat().st_mtime):
        # The C++ classes are not exported from the shared library (only the C ABIs are), so the tool is
        # linked from the same object files.
        objects = [str(p) for p in sorted(OBJ.glob("*.o"))]
        _run(["g++", *CXXFLAGS, *INCLUDES, str(src), *objects, "-o", str(MCC), "-L", str(CUDA_HOME / "lib64"),
              "-lcudart_static", "-ldl", "-lrt", "-lpthread"])
    return MCC


def build_all(force: bool = False, verbose: bool = False) -> None:
    if shutil.which("g++") is None:
        raise RuntimeError("g++ not found")
    build_library(force, verbose)
    build_mcc(force)


if __name__ == "__main__":
    ap = argparse.ArgumentParser()
    ap.add_argument("--force", action="store_true")
    args = ap.parse_args()
    build_all(args.force, verbose=True)
    print(LIB)
