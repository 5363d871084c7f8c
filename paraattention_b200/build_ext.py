"""Builds libpa_b200.so (the C-ABI CUDA library) in-tree with nvcc for sm_100a, and the small
PyTorch extension _pa_torch.so that calls it (host code only: the differentiable operators).

Run as ``python -m paraattention_b200.build_ext`` or call :func:`build`. Both are placed next to
this file so that :mod:`paraattention_b200._lib` finds them; nothing is installed outside the
source tree.
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
TORCH_EXT_PATH = PKG_DIR / "_pa_torch.so"
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


def _start_torch_ext(obj: str) -> subprocess.Popen:
    """Starts the compiler on the PyTorch extension's one source."""
    import sysconfig

    from torch.utils import cpp_extension as E

    inc = [*E.include_paths(), sysconfig.get_paths()["include"], str(Path(_nvcc()).resolve().parent.parent / "include")]
    cmd = [os.environ.get("CXX", "g++"), "-O2", "-std=c++17", "-fPIC", "-DTORCH_EXTENSION_NAME=_pa_torch",
           *[f"-I{p}" for p in inc], "-c", str(CSRC / "pa_torch.cpp"), "-o", obj]
    return subprocess.Popen(cmd, stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True)


def _link_torch_ext(obj: str) -> None:
    from torch.utils import cpp_extension as E

    libs = [p for p in E.library_paths() if Path(p).exists()]
    cmd = [os.environ.get("CXX", "g++"), "-shared", "-o", str(TORCH_EXT_PATH), obj, *[f"-L{p}" for p in libs],
           "-lc10", "-lc10_cuda", "-ltorch_cpu", "-ltorch", "-ltorch_python",
           f"-L{LIB_PATH.parent}", f"-l:{LIB_PATH.name}", "-Wl,-rpath,$ORIGIN"]
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError("linking _pa_torch.so failed:\n" + res.stdout + res.stderr)


def _stale() -> bool:
    if not LIB_PATH.exists() or not TORCH_EXT_PATH.exists():
        return True
    built = min(LIB_PATH.stat().st_mtime, TORCH_EXT_PATH.stat().st_mtime)
    deps = list(CSRC.glob("*.cpp")) + list(CSRC.glob("*.cu")) + list(CSRC.glob("*.cuh")) + list(CSRC.glob("*.h")) + list((PKG_DIR.parent / "include").glob("*.h"))
    return any(d.stat().st_mtime > built for d in deps)


def build(force: bool = False, verbose: bool = False) -> Path:
    """Compile the library and the extension if one is missing or older than its sources; return the library's path."""
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
        ext = str(Path(tmp) / "pa_torch.o")
        running.append(_start_torch_ext(ext))
        logs = [p.communicate()[0] for p in running]
        if any(p.returncode != 0 for p in running):
            raise RuntimeError("the compiler failed:\n" + "".join(log for p, log in zip(running, logs) if p.returncode != 0))
        res = subprocess.run([*cmd, "--shared", "-o", str(LIB_PATH), *objects, "-lcudart"], capture_output=True, text=True)
        if res.returncode != 0:
            raise RuntimeError("nvcc failed:\n" + res.stdout + res.stderr)
        _link_torch_ext(ext)
    if verbose:
        sys.stderr.write("".join(logs))
    return LIB_PATH


if __name__ == "__main__":
    path = build(force="--force" in sys.argv, verbose="-v" in sys.argv)
    print(path)
