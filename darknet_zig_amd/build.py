"""Builds libdkz.so, the gfx950 tensor-op library, and libdkz_dense.so, the
fused dense operators beside it, in-tree with hipcc.

Each .hip source under csrc/ (dense/) is compiled to an object for gfx950 and the
objects are linked into darknet_zig_amd/libdkz.so (libdkz_dense.so, which loads
the libdkz.so beside it). The flags are part of the
numerics: -ffp-contract=off and the correctly rounded fp32 divide/sqrt keep
every elementwise op bit-exact against the CPU twins, fp32 denormals stay
enabled as on the host, and packed-fp32 instructions are switched off.

Usage: python -m darknet_zig_amd.build [--jobs N]
"""

from __future__ import annotations

import argparse
import concurrent.futures
import os
import shutil
import subprocess
import sys
from pathlib import Path

PKG_DIR = Path(__file__).resolve().parent
REPO_DIR = PKG_DIR.parent
CSRC = PKG_DIR / "csrc"
DENSE = PKG_DIR / "dense"
INCLUDE = REPO_DIR / "include"
OBJ_DIR = PKG_DIR / "_build"
LIB_PATH = PKG_DIR / "libdkz.so"
VERSION_SCRIPT = PKG_DIR / "libdkz.map"  # exports dkz_* only
DENSE_LIB_PATH = PKG_DIR / "libdkz_dense.so"
DENSE_VERSION_SCRIPT = PKG_DIR / "libdkz_dense.map"

ARCH = "gfx950"

HIPCC_FLAGS = [
    f"--offload-arch={ARCH}",
    "-O3",
    "-std=c++17",
    "-fPIC",
    "-ffp-contract=off",
    "-fhip-fp32-correctly-rounded-divide-sqrt",
    "-fno-gpu-flush-denormals-to-zero",
    "-fno-fast-math",
    "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
    "-Wall",
    "-Wno-unused-command-line-argument",
    f"-I{INCLUDE}",
    f"-I{CSRC}",
]

# The libraries' host code: only what their header declares (visibility
# pushed to default there) is exported; the device code objects keep their
# kernels' own (protected) visibility.
VISIBILITY_FLAGS = ["-Xarch_host", "-fvisibility=hidden", "-Xarch_host", "-fvisibility-inlines-hidden"]


def hipcc() -> str:
    exe = shutil.which("hipcc") or "/opt/rocm/bin/hipcc"
    if not Path(exe).exists():
        raise RuntimeError("hipcc not found: the HIP toolchain is required to build libdkz.so")
    return exe


def sources() -> list[Path]:
    return sorted(CSRC.glob("*.hip"))


def dense_sources() -> list[Path]:
    return sorted(DENSE.glob("*.hip"))


def _compile(src: Path) -> Path:
    obj = OBJ_DIR / (("dense_" if src.parent == DENSE else "") + src.stem + ".o")
    cmd = [hipcc(), *HIPCC_FLAGS, *VISIBILITY_FLAGS, "-c", str(src), "-o", str(obj)]
    proc = subprocess.run(cmd, capture_output=True, text=True)
    if proc.returncode != 0:
        raise RuntimeError(f"hipcc failed on {src.name}:\n{proc.stdout}\n{proc.stderr}")
    return obj


def _link(lib: Path, script: Path, objs: list[Path], *extra: str) -> None:
    tmp = lib.with_suffix(".so.tmp")
    cmd = [hipcc(), f"--offload-arch={ARCH}", "-shared", "-fPIC", f"-Wl,--version-script={script}", *map(str, objs), *extra,
           "-o", str(tmp)]
    proc = subprocess.run(cmd, capture_output=True, text=True)
    if proc.returncode != 0:
        raise RuntimeError(f"linking {lib.name} failed:\n{proc.stdout}\n{proc.stderr}")
    os.replace(tmp, lib)


def build(jobs: int | None = None, verbose: bool = False) -> Path:
    """Compiles every csrc/*.hip and dense/*.hip for gfx950 and links libdkz.so and
    libdkz_dense.so. Always rebuilds."""
    OBJ_DIR.mkdir(exist_ok=True)
    srcs, dense = sources(), dense_sources()
    if not srcs or not dense:
        raise RuntimeError(f"no HIP sources under {CSRC} or {DENSE}")
    jobs = jobs or min(len(srcs) + len(dense), os.cpu_count() or 4, 8)
    with concurrent.futures.ThreadPoolExecutor(max_workers=jobs) as pool:
        objs = list(pool.map(_compile, dense + srcs))  # dense: the longest first
    _link(LIB_PATH, VERSION_SCRIPT, objs[len(dense):])
    _link(DENSE_LIB_PATH, DENSE_VERSION_SCRIPT, objs[:len(dense)], f"-L{PKG_DIR}", "-ldkz", "-Wl,-rpath,$ORIGIN")
    if verbose:
        print(f"built {LIB_PATH} and {DENSE_LIB_PATH.name} from {len(srcs) + len(dense)} sources", file=sys.stderr)
    return LIB_PATH


def main() -> None:
    ap = argparse.ArgumentParser(description=__doc__)
    ap.add_argument("--jobs", type=int, default=None)
    args = ap.parse_args()
    build(args.jobs, verbose=True)


if __name__ == "__main__":
    main()
