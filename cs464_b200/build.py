"""Ahead-of-time build of the sm_100a GEMM library `cs464_b200/libb2g.so` (nvcc, in-tree).

The reference compiles each Triton config on first use (kernels/triton_matmul.py:38-82, ~0.13 s per config, plus a
prebuilt-cubin bundle to hide it, kernels/bundle.py). Here the whole config space is one runtime-parameterised kernel,
compiled once from source by this script; first-use compile cost is zero by construction.

`python -m cs464_b200.build` rebuilds when any source or flag changed. The GEMM family's source hash is baked into the
library and returned by `b2g_source_hash()`: it covers what a stored config key compiles to (the b2g_* sources and b2g.h)
and not the microscaled operators (the micro_* sources, b2g_micro.h), so that a change there leaves stored winners valid.
"""
from __future__ import annotations

import hashlib
import os
import shutil
import subprocess
import sys
import tempfile
from concurrent.futures import ThreadPoolExecutor
from pathlib import Path

PKG = Path(__file__).resolve().parent
ROOT = PKG.parent
CSRC = PKG / "csrc"
INCLUDE = ROOT / "include"
LIB_PATH = PKG / "libb2g.so"
ARCH_FLAGS = ["-gencode", "arch=compute_100a,code=sm_100a"]
NVCC_FLAGS = ["-O3", "-lineinfo", "-std=c++17", "--expt-relaxed-constexpr", "-Xcompiler", "-fPIC,-O2", "-shared"]


def sources() -> list[Path]:
    return sorted(CSRC.glob("*.cu"))


def _hash(files: list[Path]) -> str:
    h = hashlib.sha256()
    for f in files:
        h.update(f.name.encode())
        h.update(f.read_bytes())
    h.update(" ".join(ARCH_FLAGS + NVCC_FLAGS).encode())
    return h.hexdigest()[:16]


def source_hash() -> str:
    """sha256 (16 hex) of the GEMM family's CUDA sources, headers and build flags: what a stored config key compiles to."""
    return _hash(sorted(CSRC.glob("b2g_*.cu")) + sorted(CSRC.glob("b2g_*.cuh")) + [INCLUDE / "b2g.h"])


def build_hash() -> str:
    """The same of every source in the library: whether it is up to date."""
    return _hash(sorted(CSRC.glob("*.cu")) + sorted(CSRC.glob("*.cuh")) + sorted(INCLUDE.glob("*.h")))


def nvcc() -> str:
    exe = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    if not Path(exe).exists():
        raise RuntimeError("nvcc not found: the sm_100a library cannot be built")
    return exe


def _stamp() -> Path:
    return PKG / ".libb2g.hash"


def up_to_date() -> bool:
    return LIB_PATH.exists() and _stamp().exists() and _stamp().read_text().strip() == build_hash()


def build(force: bool = False, verbose: bool = False) -> Path:
    """Compile the library for sm_100a unless it is already built from the current sources."""
    if not force and up_to_date():
        return LIB_PATH
    stamp = build_hash()
    flags = [f for f in NVCC_FLAGS if f != "-shared"] + [f"-I{INCLUDE}", f"-I{CSRC}", f'-DB2G_SOURCE_HASH="{source_hash()}"']
    if verbose:
        flags.append("-Xptxas=-v")

    def run(cmd: list[str]) -> str:
        r = subprocess.run(cmd, capture_output=True, text=True)
        if r.returncode != 0:
            raise RuntimeError(f"nvcc failed ({r.returncode}):\n{r.stdout}\n{r.stderr}")
        return r.stderr

    tmp = LIB_PATH.with_suffix(f".so.tmp{os.getpid()}")
    try:
        with tempfile.TemporaryDirectory() as d:
            objects = [str(Path(d) / (f.stem + ".o")) for f in sources()]
            cmds = [[nvcc(), *ARCH_FLAGS, *flags, "-c", str(f), "-o", o] for f, o in zip(sources(), objects)]
            if verbose:
                print("\n".join(map(" ".join, cmds)), file=sys.stderr)
            with ThreadPoolExecutor(max_workers=max(1, min(len(cmds), os.cpu_count() or 1))) as pool:
                for text in pool.map(run, cmds):
                    if verbose:
                        print(text, file=sys.stderr)
            run([nvcc(), *ARCH_FLAGS, *NVCC_FLAGS, *objects, "-o", str(tmp)])
    except BaseException:
        tmp.unlink(missing_ok=True)
        raise
    os.replace(tmp, LIB_PATH)
    _stamp().write_text(stamp + "\n")
    return LIB_PATH


if __name__ == "__main__":
    p = build(force="--force" in sys.argv, verbose="-v" in sys.argv)
    print(p)
