"""Builds libtorchft_amd.so (HIP kernels + C ABI) for gfx950 with hipcc, in-tree.

Run as ``python -m torchft_amd._build`` or call :func:`build`.  The library has
no dependency on torch: it is a plain C-ABI shared object that ctypes loads.
"""

from __future__ import annotations

import os
import shutil
import subprocess
import sys
from pathlib import Path

PKG_DIR = Path(__file__).resolve().parent
REPO_ROOT = PKG_DIR.parent
CSRC_DIR = PKG_DIR / "csrc"
SRC = CSRC_DIR / "replica_sync.hip"
ACTIVATIONS_SRC = CSRC_DIR / "activations.hip"
INCLUDE_DIR = REPO_ROOT / "include"
LIB_DIR = PKG_DIR / "lib"
LIB_PATH = LIB_DIR / "libtorchft_amd.so"
# the replica-sync source compiled with -DTFT_TUNING: additionally exports
# tft_set_launch_variant and instantiates every launch shape; loaded only by the test-suite
# and by tuning sweeps
TUNING_LIB_PATH = LIB_DIR / "libtorchft_amd_tuning.so"

# -packed-fp32-ops: keep hipcc from forming packed fp32 instructions out of the
# scalar float code (they have produced wrong results on this hardware pool).
HIPCC_FLAGS = [
    "--offload-arch=gfx950",
    "-O3",
    "-std=c++17",
    "-fPIC",
    "-Xclang",
    "-target-feature",
    "-Xclang",
    "-packed-fp32-ops",
]


def hipcc_path() -> str:
    exe = shutil.which("hipcc") or "/opt/rocm/bin/hipcc"
    if not os.path.exists(exe):
        raise RuntimeError("hipcc not found; torchft_amd needs the ROCm toolchain to build")
    return exe


def _start(args, verbose: bool) -> subprocess.Popen:
    cmd = [hipcc_path(), *args]
    if verbose:
        print("[torchft_amd] " + " ".join(cmd), flush=True)
    return subprocess.Popen(cmd, stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True)


def _finish(proc: subprocess.Popen, verbose: bool) -> None:
    stdout, _ = proc.communicate()
    # the host pass does not know the device-only feature flag; that warning is noise
    out = "\n".join(line for line in stdout.splitlines() if "packed-fp32-ops" not in line)
    if proc.returncode != 0:
        raise RuntimeError(f"hipcc failed ({proc.returncode}):\n{out}")
    if verbose and out.strip():
        print(out, flush=True)


def build(verbose: bool = True, tuning: bool = True) -> Path:
    """Compiles the library (and its tuning twin) unconditionally; returns the library's path."""
    obj_dir = LIB_DIR / "build"
    obj_dir.mkdir(parents=True, exist_ok=True)
    sync_obj, tuning_obj = obj_dir / "replica_sync.o", obj_dir / "replica_sync_tuning.o"
    activations_obj = obj_dir / "activations.o"
    sources = [(SRC, sync_obj, []), (ACTIVATIONS_SRC, activations_obj, [])]
    links = [(LIB_PATH, [sync_obj, activations_obj])]
    if tuning:
        sources.append((SRC, tuning_obj, ["-DTFT_TUNING"]))
        links.append((TUNING_LIB_PATH, [tuning_obj, activations_obj]))
    jobs = [
        _start([*HIPCC_FLAGS, *defines, f"-I{INCLUDE_DIR}", "-c", str(src), "-o", str(obj)], verbose)
        for src, obj, defines in sources
    ]
    for proc in jobs:
        _finish(proc, verbose)
    for path, objects in links:
        tmp = path.with_suffix(".so.tmp")
        _finish(_start(["--offload-arch=gfx950", "-shared", *map(str, objects), "-o", str(tmp)], verbose),
                verbose)
        os.replace(tmp, path)
    return LIB_PATH


if __name__ == "__main__":
    build()
    sys.exit(0)
