"""Build recipe for the gfx950 kernel library (and, separately, the CPU checker under oracle/).

`build_library()` cross-compiles every HIP source in `csrc/` with hipcc for gfx950 and links
`frankentorch_amd/libft_kernel_hip.so` in-tree. No GPU is needed to build. This plays the part of
the `build.rs` of an `ft-kernel-hip` crate: one hipcc invocation per translation unit, one link.
"""
from __future__ import annotations

import concurrent.futures
import os
import shutil
import subprocess
import sys

PKG_DIR = os.path.dirname(os.path.abspath(__file__))
REPO_ROOT = os.path.dirname(PKG_DIR)
CSRC = os.path.join(PKG_DIR, "csrc")
OBJ_DIR = os.path.join(PKG_DIR, "csrc", "_obj")
LIB_PATH = os.path.join(PKG_DIR, "libft_kernel_hip.so")

HIP_SOURCES = [
    "runtime.hip",
    "staging.hip",
    "stream_scratch.hip",
    "rowops.hip",
    "indexops.hip",
    "gemm.hip",
    "gemm_small.hip",
    "gemm_f64.hip",
    "gemm_split.hip",
    "sdpa.hip",
    "sdpa_decode.hip",
    "sdpa_split.hip",
    "backward.hip",
    "sdpa_bwd.hip",
    "lossops.hip",
    "ingest.hip",
    "int8ops.hip",
    "paged_append.hip",
    "paged_sdpa.hip",
    "logits.hip",
    "host_api.hip",
    "resident.hip",
]

# -ffp-contract=off: the reference never fuses a*b+c (Rust semantics), and the epilogues promise
# one rounding per step. The packed-fp32 feature is switched off because some packed forms have
# produced wrong values on this hardware.
HIPCC_FLAGS = [
    "-O3",
    "--offload-arch=gfx950",
    "-std=c++17",
    "-fPIC",
    "-ffp-contract=off",
    "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
    "-Wno-unused-command-line-argument",
]


def _hipcc() -> str:
    exe = shutil.which("hipcc") or "/opt/rocm/bin/hipcc"
    if not os.path.exists(exe):
        raise RuntimeError("hipcc not found: the gfx950 kernel library cannot be built")
    return exe


def _run(cmd: list[str]) -> None:
    proc = subprocess.run(cmd, stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True)
    out = "\n".join(l for l in proc.stdout.splitlines() if "packed-fp32-ops" not in l)
    if proc.returncode != 0:
        raise RuntimeError("command failed: %s\n%s" % (" ".join(cmd), out))
    if out.strip():
        sys.stderr.write(out + "\n")


def _compile_one(src: str) -> str:
    obj = os.path.join(OBJ_DIR, os.path.splitext(src)[0] + ".o")
    cmd = [_hipcc(), *HIPCC_FLAGS, "-I", os.path.join(REPO_ROOT, "include"), "-I", CSRC, "-c",
           os.path.join(CSRC, src), "-o", obj]
    _run(cmd)
    return obj


def build_library(jobs: int = 8) -> str:
    """Compiles and links the library; returns its path."""
    os.makedirs(OBJ_DIR, exist_ok=True)
    with concurrent.futures.ThreadPoolExecutor(max_workers=jobs) as pool:
        objs = list(pool.map(_compile_one, HIP_SOURCES))
    tmp = LIB_PATH + ".tmp"
    _run([_hipcc(), "--offload-arch=gfx950", "-shared", "-fPIC", "-o", tmp, *objs,
          "-Wl,-rpath,/opt/rocm/lib", "-Wl,--no-undefined"])
    os.replace(tmp, LIB_PATH)
    return LIB_PATH


if __name__ == "__main__":
    print(build_library())
