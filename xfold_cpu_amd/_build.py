"""Builds libxfold_hip.so in-tree (xfold_cpu_amd/lib/) with hipcc for gfx950, and the host
extension with the operators' autograd nodes beside it.

Usage: ``python -m xfold_cpu_amd._build`` (or ``__graft_entry__.build()``). Every call
recompiles; objects go to ``_build/`` at the repository root.
"""

from __future__ import annotations

import concurrent.futures
import os
import shutil
import subprocess
import sys
import sysconfig
from pathlib import Path

PACKAGE = Path(__file__).resolve().parent
ROOT = PACKAGE.parent
CSRC = PACKAGE / "csrc"
LIBDIR = PACKAGE / "lib"
OBJDIR = ROOT / "_build"
LIBRARY = LIBDIR / "libxfold_hip.so"
AUTOGRAD = LIBDIR / "xfold_autograd.so"

ARCH = "gfx950"
HIPCC = os.environ.get("HIPCC", shutil.which("hipcc") or "/opt/rocm/bin/hipcc")
# Packed fp32 VALU ops are disabled for every kernel (they have given silently wrong
# results on these boxes); hipcc's host pass warns that it does not know the feature.
FLAGS = [
    "-O3", "-std=c++17", "-fPIC", f"--offload-arch={ARCH}",
    "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
    "-Wall", "-Wno-unused-function", "-Wno-unused-variable", "-Wno-unused-result",
    f"-I{ROOT / 'include'}",
]


def sources():
    return sorted(CSRC.glob("*.hip"))


def _compile(src: Path) -> Path:
    obj = OBJDIR / (src.stem + ".o")
    cmd = [HIPCC, *FLAGS, "-c", str(src), "-o", str(obj)]
    proc = subprocess.run(cmd, capture_output=True, text=True)
    if proc.returncode != 0:
        raise RuntimeError(f"hipcc failed for {src.name}:\n{proc.stderr}")
    noisy = [line for line in proc.stderr.splitlines()
             if line.strip() and "packed-fp32-ops" not in line]
    if noisy:
        sys.stderr.write(f"[{src.name}]\n" + "\n".join(noisy) + "\n")
    return obj


def _compile_autograd() -> Path:
    """csrc/autograd.cpp: host code against torch's headers, no kernels."""
    import torch
    from torch.utils import cpp_extension

    rocm = Path(HIPCC).resolve().parent.parent
    tmp = AUTOGRAD.with_suffix(".so.tmp")
    cmd = [os.environ.get("CXX", "g++"), "-O2", "-std=c++17", "-fPIC", "-shared",
           "-DTORCH_EXTENSION_NAME=xfold_autograd", "-D__HIP_PLATFORM_AMD__=1", "-DUSE_ROCM=1",
           f"-D_GLIBCXX_USE_CXX11_ABI={int(torch.compiled_with_cxx11_abi())}",
           *(f"-isystem{path}" for path in [*cpp_extension.include_paths(), rocm / "include",
                                            sysconfig.get_paths()["include"]]),
           str(CSRC / "autograd.cpp"), "-o", str(tmp), *(f"-L{path}" for path in cpp_extension.library_paths()),
           "-lc10", "-lc10_hip", "-ltorch", "-ltorch_cpu", "-ltorch_hip", "-ltorch_python"]
    proc = subprocess.run(cmd, capture_output=True, text=True)
    if proc.returncode != 0:
        raise RuntimeError(f"{cmd[0]} failed for autograd.cpp:\n{proc.stderr}")
    os.replace(tmp, AUTOGRAD)
    return AUTOGRAD


def build(jobs: int | None = None, verbose: bool = True) -> Path:
    OBJDIR.mkdir(exist_ok=True)
    LIBDIR.mkdir(exist_ok=True)
    srcs = sources()
    jobs = jobs or min(len(srcs), max(1, min(8, os.cpu_count() or 1)))
    with concurrent.futures.ThreadPoolExecutor(max_workers=jobs) as pool:
        autograd = pool.submit(_compile_autograd)
        objs = list(pool.map(_compile, srcs))
        autograd.result()
    tmp = LIBRARY.with_suffix(".so.tmp")
    cmd = [HIPCC, f"--offload-arch={ARCH}", "-shared", "-o", str(tmp), *map(str, objs)]
    proc = subprocess.run(cmd, capture_output=True, text=True)
    if proc.returncode != 0:
        raise RuntimeError(f"link failed:\n{proc.stderr}")
    os.replace(tmp, LIBRARY)
    if verbose:
        print(f"built {LIBRARY.relative_to(ROOT)} from {len(srcs)} sources and {AUTOGRAD.relative_to(ROOT)}")
    return LIBRARY


if __name__ == "__main__":
    build()
