"""Builds ``liblazyb200.so`` in-tree with nvcc for sm_100a.

Every ``csrc/*.cu`` file is compiled to an object in ``_build/`` (in
parallel, skipped when the object is newer than its sources) and linked into
``lazy_compiler_b200/liblazyb200.so`` with the CUDA runtime linked
statically, so the library only needs the driver at run time.  The Python
side of the serving operators, ``csrc/serving_ext.cpp``, becomes the extension
module ``_serving`` beside it (against the installed torch's headers, and
again when another torch is installed).
``python -m lazy_compiler_b200.build`` runs it from the command line.
"""
from __future__ import annotations

import os
import shutil
import subprocess
import sys
from concurrent.futures import ThreadPoolExecutor
from importlib import metadata
from pathlib import Path

PACKAGE = Path(__file__).resolve().parent
ROOT = PACKAGE.parent
CSRC = PACKAGE / "csrc"
INCLUDE = ROOT / "include"
BUILD = ROOT / "_build"
LIBRARY = PACKAGE / "liblazyb200.so"
EXTENSION = PACKAGE / "_serving.so"

ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]
FLAGS = ["-O3", "-lineinfo", "-std=c++17", "-Xcompiler", "-fPIC", "--expt-relaxed-constexpr",
         "-Xptxas", "-warn-spills"]


def nvcc() -> str:
    path = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    if not Path(path).exists():
        raise RuntimeError("nvcc not found; the CUDA toolkit is required to build liblazyb200.so")
    return path


def _deps() -> list[Path]:
    return sorted(CSRC.glob("*.cuh")) + sorted(INCLUDE.glob("*.h"))


def _compile(src: Path, verbose: bool) -> Path:
    obj = BUILD / (src.stem + ".o")
    newest = max([src.stat().st_mtime] + [d.stat().st_mtime for d in _deps()])
    if obj.exists() and obj.stat().st_mtime >= newest:
        return obj
    cmd = [nvcc(), *ARCH, *FLAGS, "-I", str(INCLUDE), "-I", str(CSRC), "-c", str(src), "-o", str(obj)]
    if verbose:
        cmd[1:1] = ["-Xptxas", "-v"]
    result = subprocess.run(cmd, capture_output=True, text=True)
    if result.returncode:
        raise RuntimeError(f"nvcc failed on {src.name}:\n{result.stderr}")
    if verbose and result.stderr:
        print(result.stderr, file=sys.stderr)
    return obj


def _built_for() -> str:
    """The interpreter and the torch that the extension module is built against: its ABI is theirs."""
    try:
        return f"{sys.implementation.cache_tag} torch {metadata.version('torch')}"
    except metadata.PackageNotFoundError as e:
        raise RuntimeError("the serving operators' extension module needs torch, which is not installed") from e


def _build_extension(force: bool) -> None:
    src, stamp, built_for = CSRC / "serving_ext.cpp", BUILD / "_serving.stamp", _built_for()
    newest = max(p.stat().st_mtime for p in (src, Path(__file__), *INCLUDE.glob("*.h")))
    if EXTENSION.exists() and EXTENSION.stat().st_mtime >= newest and not force and stamp.exists() and stamp.read_text() == built_for:
        return
    import sysconfig

    import torch
    from torch.utils.cpp_extension import include_paths, library_paths
    includes = [INCLUDE, *include_paths(), Path(nvcc()).resolve().parents[1] / "include", sysconfig.get_paths()["include"]]
    tmp = EXTENSION.with_suffix(".so.tmp")
    # the libstdc++ that torch has loaded, by name: a compiler that comes with the static one only would put a second
    # copy into the module, half of its symbols shared, and writing a number to a stream then faults
    cmd = [os.environ.get("CXX", "g++"), "-O2", "-std=c++20", "-shared", "-fPIC", "-nostdlib++",
           f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}", *(f"-I{p}" for p in includes), str(src), "-o", str(tmp),
           *(f"-L{p}" for p in library_paths()), "-ltorch_python", "-ltorch", "-ltorch_cpu", "-ltorch_cuda", "-lc10_cuda", "-lc10", "-l:libstdc++.so.6"]
    result = subprocess.run(cmd, capture_output=True, text=True)
    if result.returncode:
        raise RuntimeError(f"{cmd[0]} failed on {src.name}:\n{result.stderr}")
    os.replace(tmp, EXTENSION)
    stamp.write_text(built_for)


def build(verbose: bool = False, force: bool = False) -> Path:
    """Compile every kernel source, link the shared library and the extension module; returns the library's path.

    The library needs nvcc alone: where the extension module cannot be built, it is linked before that is raised.
    """
    BUILD.mkdir(exist_ok=True)
    sources = sorted(CSRC.glob("*.cu"))
    if force:
        for obj in BUILD.glob("*.o"):
            obj.unlink()
    with ThreadPoolExecutor(max_workers=min(8, os.cpu_count() or 1)) as pool:
        extension = pool.submit(_build_extension, force)
        objects = list(pool.map(lambda s: _compile(s, verbose), sources))
    newest = max(o.stat().st_mtime for o in objects)
    if not LIBRARY.exists() or LIBRARY.stat().st_mtime < newest or force:
        tmp = LIBRARY.with_suffix(".so.tmp")
        cmd = [nvcc(), *ARCH, "-shared", "-o", str(tmp), *map(str, objects), "-cudart", "static"]
        result = subprocess.run(cmd, capture_output=True, text=True)
        if result.returncode:
            raise RuntimeError(f"link failed:\n{result.stderr}")
        os.replace(tmp, LIBRARY)
    extension.result()
    return LIBRARY


if __name__ == "__main__":
    print(build(verbose="-v" in sys.argv, force="--force" in sys.argv))
