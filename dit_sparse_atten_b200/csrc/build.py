"""Build ``libbsa.so`` (the C ABI of include/bsa.h) for sm_100a with nvcc, and
``_binding.so`` (binding.cpp: the packed operators' calls from torch) with g++.

Usage: ``python -m dit_sparse_atten_b200.csrc.build [--verbose-ptxas]``.
Both are written next to the package (``dit_sparse_atten_b200/libbsa.so``) so
they travel with the source tree; each is rebuilt only when a source is newer.
"""

from __future__ import annotations

import argparse
import os
import shutil
import subprocess
import sys
from concurrent.futures import ThreadPoolExecutor
from pathlib import Path

CSRC = Path(__file__).resolve().parent
PACKAGE = CSRC.parent
REPO = PACKAGE.parent
LIBRARY = PACKAGE / "libbsa.so"
BINDING = PACKAGE / "_binding.so"
SOURCES = sorted(CSRC.glob("*.cu"))
HEADERS = sorted(CSRC.glob("*.cuh")) + sorted(CSRC.glob("*.h")) + [REPO / "include" / "bsa.h"]

NVCC_FLAGS = [
    "-gencode", "arch=compute_100a,code=sm_100a",
    "-O3", "-lineinfo", "-std=c++17",
    "-Xcompiler", "-fPIC", "-Xcompiler", "-fvisibility=hidden",
    "--expt-relaxed-constexpr",
    "-I", str(REPO / "include"),
]


def nvcc_path() -> str:
    for candidate in (os.environ.get("NVCC"), shutil.which("nvcc"), "/usr/local/cuda/bin/nvcc"):
        if candidate and Path(candidate).exists():
            return candidate
    raise RuntimeError("nvcc not found; the CUDA toolkit is required to build libbsa.so")


def up_to_date() -> bool:
    if not LIBRARY.exists():
        return False
    built = LIBRARY.stat().st_mtime
    return all(p.stat().st_mtime <= built for p in SOURCES + HEADERS if p.exists())


def build(force: bool = False, verbose_ptxas: bool = False) -> Path:
    if not force and up_to_date():
        return LIBRARY
    nvcc = nvcc_path()
    objdir = REPO / "_build"
    objdir.mkdir(exist_ok=True)
    objects, commands = [], []
    for src in SOURCES:
        obj = objdir / (src.stem + ".o")
        cmd = [nvcc, *NVCC_FLAGS, "-c", str(src), "-o", str(obj)]
        if verbose_ptxas:
            cmd[1:1] = ["-Xptxas", "-v"]
        commands.append(cmd)
        objects.append(str(obj))
    # one nvcc per translation unit, in parallel
    with ThreadPoolExecutor(max_workers=min(len(commands), os.cpu_count() or 1)) as pool:
        for done in pool.map(lambda c: subprocess.run(c, capture_output=True, text=True),
                             commands):
            sys.stdout.write(done.stdout)
            sys.stderr.write(done.stderr)
            done.check_returncode()
    tmp = LIBRARY.with_suffix(".so.tmp")
    subprocess.run([nvcc, "-shared", "-gencode", "arch=compute_100a,code=sm_100a",
                    "-o", str(tmp), *objects], check=True)
    os.replace(tmp, LIBRARY)
    return LIBRARY


def binding_up_to_date() -> bool:
    import torch

    from .._native import binding_torch_version

    if binding_torch_version(BINDING) != str(torch.__version__):
        return False
    sources = [CSRC / "binding.cpp", REPO / "include" / "bsa.h", Path(__file__)]
    return all(p.stat().st_mtime <= BINDING.stat().st_mtime for p in sources)


def build_binding(force: bool = False) -> Path:
    """``_binding.so``; the entry points of ``libbsa.so`` are handed to it at run time."""
    if not force and binding_up_to_date():
        return BINDING
    import sysconfig

    import torch
    from torch.utils import cpp_extension

    includes = cpp_extension.include_paths("cuda") + [sysconfig.get_paths()["include"]]
    torch_lib = str(Path(torch.__file__).resolve().parent / "lib")
    tmp = BINDING.with_suffix(".so.tmp")
    cmd = ["g++", "-O2", "-std=c++17", "-fPIC", "-shared", "-fvisibility=hidden",
           f'-DBSA_TORCH_VERSION="{torch.__version__}"',
           f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
           *[f"-I{p}" for p in includes], str(CSRC / "binding.cpp"), "-o", str(tmp),
           f"-L{torch_lib}", "-ltorch_python", "-ltorch", "-ltorch_cpu", "-lc10", "-lc10_cuda"]
    done = subprocess.run(cmd, capture_output=True, text=True)
    sys.stderr.write(done.stderr)
    done.check_returncode()
    os.replace(tmp, BINDING)
    return BINDING


def main(argv=None) -> int:
    parser = argparse.ArgumentParser(description=__doc__)
    parser.add_argument("--force", action="store_true")
    parser.add_argument("--verbose-ptxas", action="store_true")
    args = parser.parse_args(argv)
    print(build(force=args.force, verbose_ptxas=args.verbose_ptxas))
    print(build_binding(force=args.force))
    return 0


if __name__ == "__main__":
    sys.exit(main())
