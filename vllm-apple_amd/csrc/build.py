"""Build libvllm_apple_amd.so for gfx950 with hipcc.

Each .hip file is compiled to an object in parallel, then linked into one
shared library placed next to the Python package, in-tree, so it ships with
the source tree.  Run directly (``python build.py``) or through
``vllm_apple_amd.build_library()``.
"""
from __future__ import annotations

import concurrent.futures as cf
import os
import shutil
import subprocess
import sys
from pathlib import Path

HERE = Path(__file__).resolve().parent
PKG_ROOT = HERE.parent                      # vllm-apple_amd/
REPO = PKG_ROOT.parent                      # repository root
INCLUDE = REPO / "include"
OUT_DIR = PKG_ROOT / "vllm_apple_amd"
LIB_NAME = "libvllm_apple_amd.so"
OBJ_DIR = PKG_ROOT / "_build"
HOST_NAME = "_host.so"                      # the Python extension (host_calls.cpp)

SOURCES = [
    "status.hip",
    "kv_write.hip",
    "paged_decode.hip",
    "paged_prefill.hip",
    "layer_ops.hip",
    "index_ops.hip",
    "qkv_epilogue.hip",
    "topk.hip",
    "gate_up_silu.hip",
    "kv_stream.hip",
    "kv_quant.hip",
    "decode_view.hip",
    "prefill_view.hip",
]

ARCH = os.environ.get("VAA_OFFLOAD_ARCH", "gfx950")

# Per-source flags.  The prefill kernel's row maxima take fmaxf over MFMA
# results; under IEEE NaN rules each operand is first canonicalised (one extra
# v_max_f32 per score).  Scores are finite or the -inf of a masked key, so
# the kernel is built without NaN semantics (infinities are kept): 3.5 %
# faster on C3.
#
# The prefill over a vaa_kv_view is built the same way, for the same reason.
#
# The gate/up GEMM and the prefills issue their direct-to-LDS loads as inline
# asm that writes M0; clang warns that M0 is reserved because
# compiler-generated code may use it (the asm declares it clobbered).
FILE_FLAGS = {
    "paged_prefill.hip": ["-fno-honor-nans", "-Wno-inline-asm"],
    "prefill_view.hip": ["-fno-honor-nans", "-Wno-inline-asm"],
    "gate_up_silu.hip": ["-Wno-inline-asm"],
}


def hipcc() -> str:
    for cand in (os.environ.get("HIPCC"), "/opt/rocm/bin/hipcc", shutil.which("hipcc")):
        if cand and Path(cand).exists():
            return cand
    raise RuntimeError("hipcc not found (set HIPCC or install ROCm)")


def common_flags() -> list[str]:
    return [
        f"--offload-arch={ARCH}",
        "-O3",
        "-std=c++17",
        "-fPIC",
        "-Wall",
        "-Wno-unused-function",
        f"-I{INCLUDE}",
        f"-I{HERE}",
        # Keep hipcc from emitting packed-fp32 VALU ops.
        "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
    ]


def _compile(src: str) -> Path:
    obj = OBJ_DIR / (Path(src).stem + ".o")
    cmd = [hipcc(), *common_flags(), *FILE_FLAGS.get(src, []), "-c", str(HERE / src), "-o",
           str(obj)]
    res = subprocess.run(cmd, capture_output=True, text=True)
    noise = "is not a recognized feature for this target"
    err = "\n".join(l for l in res.stderr.splitlines() if noise not in l)
    if res.returncode != 0:
        raise RuntimeError(f"hipcc failed for {src}:\n{err}")
    if err.strip():
        sys.stderr.write(err + "\n")
    return obj


def build_host() -> Path:
    """The wrappers' native host path: a CPython extension over torch's C++
    headers, plain host code."""
    import sysconfig

    import torch
    from torch.utils.cpp_extension import include_paths, library_paths

    out = OUT_DIR / HOST_NAME
    tmp = OBJ_DIR / (HOST_NAME + ".tmp")
    cxx = os.environ.get("CXX") or shutil.which("g++") or hipcc()
    cmd = [cxx, "-O2", "-std=c++17", "-fPIC", "-shared", "-Wall",
           f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
           f"-I{INCLUDE}", f"-I{sysconfig.get_paths()['include']}",
           *(f"-isystem{d}" for d in include_paths()), str(HERE / "host_calls.cpp"),
           "-o", str(tmp), *(f"-L{d}" for d in library_paths()),
           "-ltorch_python", "-ltorch_cpu", "-lc10", "-ldl"]
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError(f"{cxx} failed for host_calls.cpp:\n{res.stderr}")
    os.replace(tmp, out)
    return out


def build(verbose: bool = True) -> Path:
    OBJ_DIR.mkdir(parents=True, exist_ok=True)
    with cf.ThreadPoolExecutor(max_workers=min(len(SOURCES), os.cpu_count() or 4)) as ex:
        host = ex.submit(build_host)
        objs = list(ex.map(_compile, SOURCES))
        host.result()
    out = OUT_DIR / LIB_NAME
    tmp = out.with_suffix(".so.tmp")
    cmd = [hipcc(), f"--offload-arch={ARCH}", "-shared", "-fPIC", *map(str, objs), "-o", str(tmp)]
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError(f"link failed:\n{res.stderr}")
    os.replace(tmp, out)
    if verbose:
        print(f"built {out}")
    return out


if __name__ == "__main__":
    build()
