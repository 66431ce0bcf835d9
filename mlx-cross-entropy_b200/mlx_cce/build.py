"""Compile the sources of this package in-tree: ``libcce_b200.so`` (CUDA) and
``libcce_torch.so`` (the torch operators that call it).

The library is built for sm_100a only (``-gencode arch=compute_100a,code=sm_100a``)
with nvcc; it links the CUDA runtime statically and resolves the driver's
tensor-map encoder at run time, so it loads on a machine without a GPU and
needs nothing at run time but the NVIDIA driver.  The torch operators are host
code (g++, torch's own headers) and belong to the torch they were built with.

    python mlx-cross-entropy_b200/mlx_cce/build.py           # rebuild if stale
    python mlx-cross-entropy_b200/mlx_cce/build.py --force

(Run it as a script: importing the package itself loads the library.)
"""

from __future__ import annotations

import os
import shutil
import subprocess
import sys
from pathlib import Path

PKG_DIR = Path(__file__).resolve().parent
ROOT = PKG_DIR.parent                     # mlx-cross-entropy_b200/
CSRC = ROOT / "csrc"
REPO = ROOT.parent
INCLUDE = REPO / "include"
LIB_NAME = "libcce_b200.so"
LIB_PATH = PKG_DIR / LIB_NAME
TORCH_SOURCE = CSRC / "torch_ops.cpp"
TORCH_LIB_PATH = PKG_DIR / "libcce_torch.so"

SOURCES = ["cce_abi.cu", "aux_kernels.cu", "simt_kernels.cu", "tc_kernels.cu", "noalloc.cu", "peer.cu",
           "token_loss.cu", "rows_kernels.cu"]

NVCC_FLAGS = [
    "-gencode", "arch=compute_100a,code=sm_100a",
    "-O3", "-lineinfo", "-std=c++17",
    "-Xcompiler", "-fPIC,-O3,-fvisibility=hidden",
    "--expt-relaxed-constexpr",
    "-shared",
]


def nvcc_path() -> str:
    for cand in (os.environ.get("NVCC"), shutil.which("nvcc"), "/usr/local/cuda/bin/nvcc"):
        if cand and Path(cand).exists():
            return cand
    raise RuntimeError("nvcc not found: set $NVCC or put the CUDA toolkit on PATH")


def _deps():
    deps = [CSRC / s for s in SOURCES]
    deps += sorted(CSRC.glob("*.cuh"))
    deps += sorted(INCLUDE.glob("*.h"))
    return deps


def _stale(lib: Path, deps) -> bool:
    if not lib.exists():
        return True
    t = lib.stat().st_mtime
    return any(p.stat().st_mtime > t for p in deps)


def needs_build() -> bool:
    return _stale(LIB_PATH, _deps())


def _run(cmd, what, verbose):
    if verbose:
        print(" ".join(cmd), file=sys.stderr)
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError(f"{what} failed ({res.returncode}):\n{res.stdout}\n{res.stderr}")


# Text in the torch operators' library, followed by the version of the torch that it was built for.
_BUILT_FOR = b"cce_b200 operators for torch "


def torch_built_for(path: Path = TORCH_LIB_PATH):
    """The version of torch that the operators at ``path`` were built for (None: it does not say)."""
    data = path.read_bytes()
    at = data.find(_BUILT_FOR)
    return None if at < 0 else data[at + len(_BUILT_FOR):data.index(b"\0", at)].decode()


def build_torch_ops(force: bool = False, verbose: bool = False) -> Path:
    """Compile the torch operators if missing, stale or of another torch; return their path."""
    import torch
    if not force and not _stale(TORCH_LIB_PATH, [TORCH_SOURCE, *INCLUDE.glob("*.h")]) \
            and torch_built_for() == torch.__version__:
        return TORCH_LIB_PATH
    home = Path(torch.__file__).resolve().parent
    cuda = Path(nvcc_path()).resolve().parent.parent
    tmp = TORCH_LIB_PATH.with_suffix(".so.tmp")
    cmd = [os.environ.get("CXX") or "g++", "-std=c++17", "-O2", "-fPIC", "-shared", "-fvisibility=hidden",
           f"-D_GLIBCXX_USE_CXX11_ABI={int(torch.compiled_with_cxx11_abi())}",
           f'-DCCE_BUILT_FOR="{_BUILT_FOR.decode()}{torch.__version__}"', f"-I{INCLUDE}", f"-I{home / 'include'}",
           f"-I{home / 'include' / 'torch' / 'csrc' / 'api' / 'include'}", f"-I{cuda / 'include'}", str(TORCH_SOURCE),
           "-o", str(tmp), f"-L{home / 'lib'}", "-ltorch_cpu", "-lc10", "-lc10_cuda"]
    _run(cmd, "g++", verbose)
    os.replace(tmp, TORCH_LIB_PATH)
    return TORCH_LIB_PATH


def build(force: bool = False, verbose: bool = False) -> Path:
    """Compile the shared libraries if missing or stale; return the CUDA library's path."""
    if force or needs_build():
        tmp = LIB_PATH.with_suffix(".so.tmp")
        cmd = [nvcc_path(), *NVCC_FLAGS, f"-I{INCLUDE}", f"-I{CSRC}", "-o", str(tmp)]
        cmd += [str(CSRC / s) for s in SOURCES]
        _run(cmd, "nvcc", verbose)
        os.replace(tmp, LIB_PATH)
    build_torch_ops(force, verbose)
    return LIB_PATH


if __name__ == "__main__":
    p = build(force="--force" in sys.argv, verbose=True)
    print(p)
