"""Build recipe for the sm_100a shared library (``libfreemoe_b200.so``), which
needs nvcc alone, and the entry points for torch tensors beside it
(``_torch_calls.<python>.torch-<version>.so``), where torch is installed.

The library is built in-tree with nvcc so that the ``.so`` travels with the
source tree; nothing is JIT-compiled or installed into site-packages.
"""
from __future__ import annotations

import os
import subprocess
import sys
from concurrent.futures import ThreadPoolExecutor
from pathlib import Path

PKG = Path(__file__).resolve().parent
ROOT = PKG.parent
CSRC = PKG / "csrc"
INCLUDE = ROOT / "include"
LIB = PKG / "libfreemoe_b200.so"

ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]
NVCC_FLAGS = [
    "-O3", "-std=c++17", "-lineinfo", "--expt-relaxed-constexpr",
    "-Xcompiler", "-fPIC", "-Xcompiler", "-Wall",
    "-Xptxas", "-warn-spills",
]


def nvcc() -> str:
    cand = os.environ.get("NVCC") or "/usr/local/cuda/bin/nvcc"
    return cand if Path(cand).exists() else "nvcc"


def sources() -> list[Path]:
    return sorted(CSRC.glob("*.cu"))


def _stale(target: Path, deps: list[Path]) -> bool:
    if not target.exists():
        return True
    t = target.stat().st_mtime
    return any(d.stat().st_mtime > t for d in deps)


def torch_calls_path() -> Path:
    """The build of the entry points for this Python and this torch: another's is never loaded."""
    import torch

    return PKG / f"_torch_calls.{sys.implementation.cache_tag}.torch-{torch.__version__}.so"


def build_torch_calls(force: bool = False, verbose: bool = False) -> Path | None:
    """Compiles ``csrc/torch_calls.cpp``, the entry points for torch tensors, against the
    installed torch (host code only: it calls the library through the addresses it is given).
    Without a torch there are none, and nothing here needs them."""
    try:
        target = torch_calls_path()
    except ImportError:
        print("torch is not installed: the library is built without entry points for its tensors", file=sys.stderr)
        return None
    src = CSRC / "torch_calls.cpp"
    if not force and not _stale(target, [src, Path(__file__), *INCLUDE.glob("*.h")]):
        return target
    import sysconfig

    import torch
    from torch.utils import cpp_extension

    lib = Path(torch.__file__).resolve().parent / "lib"
    include = [*cpp_extension.include_paths(), sysconfig.get_paths()["include"], "/usr/local/cuda/include", str(INCLUDE)]
    tmp = target.with_suffix(".so.tmp")
    cmd = ["g++", "-O2", "-std=c++17", "-fPIC", "-shared", "-fvisibility=hidden", "-DTORCH_EXTENSION_NAME=_torch_calls",
           f"-D_GLIBCXX_USE_CXX11_ABI={int(torch.compiled_with_cxx11_abi())}", *(f"-I{i}" for i in include), str(src),
           f"-L{lib}", "-ltorch_python", "-ltorch", "-ltorch_cpu", "-lc10", "-lc10_cuda", f"-Wl,-rpath,{lib}",
           "-o", str(tmp)]
    if verbose:
        print(" ".join(cmd), file=sys.stderr)
    subprocess.run(cmd, check=True)
    os.replace(tmp, target)
    return target


def build(force: bool = False, verbose: bool = False, ptxas_verbose: bool = False) -> Path:
    """The library, and meanwhile the entry points for torch tensors; what fails in these is
    raised when the library is there."""
    with ThreadPoolExecutor(1) as pool:
        calls = pool.submit(build_torch_calls, force, verbose)
        lib = build_library(force, verbose, ptxas_verbose)
        calls.result()
    return lib


def build_library(force: bool = False, verbose: bool = False, ptxas_verbose: bool = False) -> Path:
    """Compiles every ``csrc/*.cu`` for sm_100a into ``libfreemoe_b200.so``."""
    deps = sources() + sorted(CSRC.glob("*.cuh")) + sorted(INCLUDE.glob("*.h")) + [Path(__file__)]
    if not force and not _stale(LIB, deps):
        return LIB
    objdir = PKG / "_build"
    objdir.mkdir(exist_ok=True)
    objs = []
    procs = []
    for src in sources():
        obj = objdir / (src.stem + ".o")
        cmd = [nvcc(), *ARCH, *NVCC_FLAGS, "-I", str(INCLUDE), "-I", str(CSRC), "-c", str(src), "-o", str(obj)]
        if ptxas_verbose:
            cmd[1:1] = ["-Xptxas", "-v"]
        if verbose:
            print(" ".join(cmd), file=sys.stderr)
        procs.append((src, subprocess.Popen(cmd, stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True)))
        objs.append(obj)
    failed = []
    for src, p in procs:
        out, _ = p.communicate()
        if out and (verbose or ptxas_verbose or p.returncode):
            print(out, file=sys.stderr)
        if p.returncode:
            failed.append(src.name)
    if failed:
        raise RuntimeError(f"nvcc failed for: {', '.join(failed)}")
    tmp = LIB.with_suffix(".so.tmp")
    # --no-undefined: a symbol missing from every object fails the build here,
    # not the first dlopen on a GPU box
    link = [nvcc(), *ARCH, "-shared", "-Xcompiler", "-fPIC", "-Xlinker", "--no-undefined", *map(str, objs),
            "-o", str(tmp)]
    if verbose:
        print(" ".join(link), file=sys.stderr)
    subprocess.run(link, check=True)
    os.replace(tmp, LIB)
    return LIB


if __name__ == "__main__":
    build(force="--force" in sys.argv, verbose="-v" in sys.argv, ptxas_verbose="--ptxas" in sys.argv)
    print(LIB)
