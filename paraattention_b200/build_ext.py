"""Builds libpa_b200.so (the C-ABI CUDA library) in-tree with nvcc for sm_100a.

Run as ``python -m paraattention_b200.build_ext`` or call :func:`build`. The library is
placed next to this file so that :mod:`paraattention_b200._lib` finds it; nothing is
installed outside the source tree.
"""
from __future__ import annotations

import os
import shutil
import subprocess
import sys
import tempfile
from pathlib import Path

PKG_DIR = Path(__file__).resolve().parent
CSRC = PKG_DIR / "csrc"
LIB_PATH = PKG_DIR / "libpa_b200.so"
SOURCES = ["pa_api.cu", "pa_qk_norm.cu", "pa_xattn_fwd.cu", "pa_xattn_bwd.cu"]
NVCC_FLAGS = [
    "-gencode", "arch=compute_100a,code=sm_100a",
    "-lineinfo", "-O3", "-std=c++17",
    "-Xcompiler", "-fPIC",
]


def _nvcc() -> str:
    cand = os.environ.get("NVCC") or shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    if not Path(cand).exists():
        raise RuntimeError("nvcc not found; set NVCC or add it to PATH")
    return cand


def _stale() -> bool:
    if not LIB_PATH.exists():
        return True
    built = LIB_PATH.stat().st_mtime
    deps = list(CSRC.glob("*.cu")) + list(CSRC.glob("*.cuh")) + list(CSRC.glob("*.h")) + list((PKG_DIR.parent / "include").glob("*.h"))
    return any(d.stat().st_mtime > built for d in deps)


def build(force: bool = False, verbose: bool = False) -> Path:
    """Compile the library if it is missing or older than its sources; return its path."""
    if not force and not _stale():
        return LIB_PATH
    cmd = [_nvcc(), *NVCC_FLAGS]
    if verbose:
        cmd += ["-Xptxas", "-v"]
    with tempfile.TemporaryDirectory() as tmp:
        # one compiler per source, all at once: each takes most of a minute
        objects = [str(Path(tmp) / (Path(src).stem + ".o")) for src in SOURCES]
        running = [subprocess.Popen([*cmd, "-c", "-o", obj, str(CSRC / src)], stdout=subprocess.PIPE,
                                    stderr=subprocess.STDOUT, text=True) for src, obj in zip(SOURCES, objects)]
        logs = [p.communicate()[0] for p in running]
        if any(p.returncode != 0 for p in running):
            raise RuntimeError("nvcc failed:\n" + "".join(log for p, log in zip(running, logs) if p.returncode != 0))
        res = subprocess.run([*cmd, "--shared", "-o", str(LIB_PATH), *objects, "-lcudart"], capture_output=True, text=True)
        if res.returncode != 0:
            raise RuntimeError("nvcc failed:\n" + res.stdout + res.stderr)
    if verbose:
        sys.stderr.write("".join(logs))
    return LIB_PATH


if __name__ == "__main__":
    path = build(force="--force" in sys.argv, verbose="-v" in sys.argv)
    print(path)
