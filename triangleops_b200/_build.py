"""Build recipe for the in-tree C-ABI library ``libtriangleops_b200.so`` and the
Python extension ``_bind.so`` on top of it.

The whole CUDA side is one translation unit (``csrc/tops_all.cu``) compiled for
sm_100a only. ``nvcc`` cross-compiles without a GPU, so this runs anywhere the
CUDA toolkit is installed; the resulting ``.so`` sits next to this file and is
loaded with ``ctypes`` by :mod:`triangleops_b200._lib`. The extension
(``csrc/bind.cpp``, host code only, against torch's headers) holds the launchers
of the token block's operators.
"""

from __future__ import annotations

import os
import shutil
import subprocess
import sys

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
LIB_NAME = "libtriangleops_b200.so"
LIB_PATH = os.path.join(HERE, LIB_NAME)
BIND_SRC = os.path.join(CSRC, "bind.cpp")
BIND_PATH = os.path.join(HERE, "_bind.so")
BIND_STAMP = BIND_PATH + ".for"  # what _bind.so was compiled against

NVCC_FLAGS = [
    "-gencode",
    "arch=compute_100a,code=sm_100a",
    "-O3",
    "-lineinfo",
    "-std=c++17",
    "-Xcompiler",
    "-fPIC",
    "-shared",
    "--expt-relaxed-constexpr",
]


def _nvcc() -> str:
    for cand in (os.environ.get("NVCC"), shutil.which("nvcc"), "/usr/local/cuda/bin/nvcc"):
        if cand and os.path.exists(cand):
            return cand
    raise RuntimeError("nvcc not found; the CUDA toolkit is required to build triangleops_b200")


def _sources() -> list[str]:
    out = []
    for root, _, files in os.walk(CSRC):
        for f in files:
            if f.endswith((".cu", ".cuh", ".h")):
                out.append(os.path.join(root, f))
    return out


def needs_build() -> bool:
    if not os.path.exists(LIB_PATH):
        return True
    t = os.path.getmtime(LIB_PATH)
    return any(os.path.getmtime(s) > t for s in _sources())


def _bind_against() -> str:
    import torch

    return f"torch {torch.__version__}, Python {sys.version_info.major}.{sys.version_info.minor}"


def needs_bind() -> bool:
    """Whether ``_bind.so`` is missing, older than its sources, or of another torch or Python than
    this process's (whose C++ interfaces it would call as if they were its own)."""
    if not os.path.exists(BIND_PATH) or not os.path.exists(BIND_STAMP):
        return True
    with open(BIND_STAMP) as f:
        if f.read() != _bind_against():
            return True
    header = os.path.join(HERE, "..", "include", "triangleops_b200.h")
    t = os.path.getmtime(BIND_PATH)
    return any(os.path.exists(s) and os.path.getmtime(s) > t for s in (BIND_SRC, os.path.join(CSRC, "status.h"), header))


def _run(cmd: list[str], tmp: str, path: str, verbose: bool) -> None:
    if verbose:
        print(" ".join(cmd), file=sys.stderr)
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError(f"{cmd[0]} failed ({res.returncode}):\n{res.stdout}\n{res.stderr}")
    os.replace(tmp, path)


def build_bind(verbose: bool = False, force: bool = False) -> str:
    """Compile ``csrc/bind.cpp`` into ``_bind.so``, linked to ``libtriangleops_b200.so``."""
    build(verbose=verbose)
    if not force and not needs_bind():
        return BIND_PATH
    import sysconfig

    import torch

    root = os.path.dirname(torch.__file__)
    cuda = os.environ.get("CUDA_HOME") or os.path.dirname(os.path.dirname(_nvcc()))
    tmp = f"{BIND_PATH}.{os.getpid()}.tmp"
    inc = (os.path.join(root, "include"), os.path.join(root, "include", "torch", "csrc", "api", "include"),
           os.path.join(cuda, "include"), sysconfig.get_paths()["include"])
    cmd = [os.environ.get("CXX") or shutil.which("g++") or "g++", "-O2", "-std=c++17", "-shared", "-fPIC", "-w",
           f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}", *(f"-I{d}" for d in inc), BIND_SRC, "-o",
           tmp, f"-L{HERE}", f"-l:{LIB_NAME}", f"-L{os.path.join(root, 'lib')}", "-ltorch_python", "-ltorch",
           "-ltorch_cpu", "-ltorch_cuda", "-lc10", "-lc10_cuda", "-Wl,-rpath,$ORIGIN"]
    _run(cmd, tmp, BIND_PATH, verbose)
    with open(tmp, "w") as f:
        f.write(_bind_against())
    os.replace(tmp, BIND_STAMP)
    return BIND_PATH


def build(verbose: bool = False, force: bool = False, extra_flags: list[str] | None = None) -> str:
    """Compile ``csrc/tops_all.cu`` into ``libtriangleops_b200.so`` (sm_100a)."""
    if not force and not needs_build():
        return LIB_PATH
    tmp = f"{LIB_PATH}.{os.getpid()}.tmp"
    cmd = [_nvcc(), *NVCC_FLAGS, *(extra_flags or []), os.path.join(CSRC, "tops_all.cu"), "-o", tmp]
    _run(cmd, tmp, LIB_PATH, verbose)
    return LIB_PATH


if __name__ == "__main__":
    print(build(verbose=True, force="--force" in sys.argv))
    print(build_bind(verbose=True, force="--force" in sys.argv))
