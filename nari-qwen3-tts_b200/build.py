"""Build recipe for libnqt.so, the sm_100a kernels behind include/nqt.h, and
for _nqt_bind.so, the Python entry of the 8-bit operators.

Every ``csrc/*.cu`` file is compiled with nvcc for ``sm_100a`` only and the
objects are linked into ``libnqt.so`` next to this file (in-tree, so the
library travels with the source tree).  Objects go to ``_build/``.
``csrc/bind.cpp`` is compiled with the host compiler against the running
Python and torch.  A rebuild happens only when a source or header is newer
than the libraries, or when the binding was compiled against another Python
or torch.
"""

from __future__ import annotations

import concurrent.futures
import os
import shutil
import subprocess
import sysconfig
from pathlib import Path

PKG_DIR = Path(__file__).resolve().parent
REPO_DIR = PKG_DIR.parent
CSRC = PKG_DIR / "csrc"
BUILD_DIR = PKG_DIR / "_build"
LIB_PATH = PKG_DIR / "libnqt.so"
BIND_PATH = PKG_DIR / "_nqt_bind.so"

ARCH_FLAGS = ["-gencode", "arch=compute_100a,code=sm_100a"]
NVCC_FLAGS = [
    *ARCH_FLAGS,
    "-lineinfo",
    "-O3",
    "-std=c++17",
    "-Xcompiler",
    "-fPIC",
    "--expt-relaxed-constexpr",
    f"-I{REPO_DIR / 'include'}",
]


def _nvcc() -> str:
    for candidate in (os.environ.get("NVCC"), shutil.which("nvcc"), "/usr/local/cuda/bin/nvcc"):
        if candidate and Path(candidate).exists():
            return candidate
    raise RuntimeError("nvcc not found: set NVCC or put the CUDA toolkit on PATH")


def sources() -> list[Path]:
    return sorted(CSRC.glob("*.cu"))


def _inputs() -> list[Path]:
    return [*sources(), *CSRC.glob("*.cuh"), *(REPO_DIR / "include").glob("*.h")]


def _newer(target: Path, inputs: list[Path]) -> bool:
    return target.exists() and all(p.stat().st_mtime <= target.stat().st_mtime for p in inputs)


def up_to_date() -> bool:
    return _newer(LIB_PATH, _inputs()) and _bind_up_to_date()


def _bind_key() -> str:
    """What the binding was compiled against, besides its sources."""

    import torch

    return f"{sysconfig.get_config_var('SOABI')} torch {torch.__version__}"


def _bind_stamp() -> Path:
    return BUILD_DIR / "bind.txt"


def _mark_bind() -> None:
    _bind_stamp().write_text(_bind_key())


def _bind_up_to_date() -> bool:
    return (_newer(BIND_PATH, [CSRC / "bind.cpp", *(REPO_DIR / "include").glob("*.h")]) and _bind_stamp().exists()
            and _bind_stamp().read_text() == _bind_key())


def _cuda_include() -> Path:
    return Path(_nvcc()).resolve().parent.parent / "include"


def build_bind() -> Path:
    """Compile the Python entry of the 8-bit operators against torch's headers."""

    import torch

    root = Path(torch.__path__[0])
    tmp = BIND_PATH.with_suffix(".so.tmp")
    cmd = [
        os.environ.get("CXX", "g++"), "-O2", "-std=c++17", "-shared", "-fPIC",
        f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
        f"-I{root / 'include'}", f"-I{root / 'include/torch/csrc/api/include'}",
        f"-I{sysconfig.get_paths()['include']}", f"-I{_cuda_include()}",
        str(CSRC / "bind.cpp"), "-o", str(tmp), f"-L{root / 'lib'}",
        "-lc10", "-lc10_cuda", "-ltorch_cpu", "-ltorch", "-ltorch_python",
    ]
    proc = subprocess.run(cmd, capture_output=True, text=True)
    if proc.returncode != 0:
        raise RuntimeError(f"compiling bind.cpp failed:\n{proc.stderr}")
    os.replace(tmp, BIND_PATH)
    BUILD_DIR.mkdir(exist_ok=True)
    _mark_bind()
    return BIND_PATH


def build(*, force: bool = False, verbose: bool = False) -> Path:
    """Compile all kernels and link libnqt.so; returns the library path."""

    if not force and up_to_date():
        return LIB_PATH
    nvcc = _nvcc()
    BUILD_DIR.mkdir(exist_ok=True)

    def compile_one(src: Path) -> Path:
        obj = BUILD_DIR / (src.stem + ".o")
        cmd = [nvcc, *NVCC_FLAGS, "-c", str(src), "-o", str(obj)]
        if verbose:
            cmd.insert(1, "-Xptxas=-v")
        proc = subprocess.run(cmd, capture_output=True, text=True)
        if proc.returncode != 0:
            raise RuntimeError(f"nvcc failed for {src.name}:\n{proc.stderr}")
        if verbose and proc.stderr:
            print(proc.stderr)
        return obj

    with concurrent.futures.ThreadPoolExecutor(max_workers=min(8, os.cpu_count() or 1)) as pool:
        bind = pool.submit(build_bind) if force or not _bind_up_to_date() else None
        objects = list(pool.map(compile_one, sources()))
        if bind is not None:
            bind.result()
    tmp = LIB_PATH.with_suffix(".so.tmp")
    cmd = [nvcc, *ARCH_FLAGS, "-shared", "-o", str(tmp), *map(str, objects)]
    proc = subprocess.run(cmd, capture_output=True, text=True)
    if proc.returncode != 0:
        raise RuntimeError(f"link of libnqt.so failed:\n{proc.stderr}")
    os.replace(tmp, LIB_PATH)
    return LIB_PATH


if __name__ == "__main__":
    import sys

    print(build(force="--force" in sys.argv, verbose="-v" in sys.argv))
