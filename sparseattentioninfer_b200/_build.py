"""Build the in-tree C-ABI library ``_lib/libsa_b200.so`` with nvcc for sm_100a, and
``_lib/_sa_paged-*.so``, the compiled Python binding of the paged-cache operators.

The library is plain CUDA C++ (no torch headers), so it builds without a GPU and
loads in any process through ctypes; the binding is host C++ against the headers
of the installed torch and Python, whose versions its file name carries. Run
``python sparseattentioninfer_b200/_build.py`` (as a file: importing the package
itself requires the built library).
"""
from __future__ import annotations

import importlib.metadata
import importlib.util
import os
import shutil
import subprocess
import sys
import sysconfig
from pathlib import Path

PKG = Path(__file__).resolve().parent
CSRC = PKG / "csrc"
LIB_DIR = PKG / "_lib"
LIB_PATH = LIB_DIR / "libsa_b200.so"
INCLUDE = PKG.parent / "include"
BINDING_SRC = CSRC / "paged_binding.cpp"

ARCH_FLAGS = ["-gencode", "arch=compute_100a,code=sm_100a"]
BASE_FLAGS = [
    "-O3",
    "-std=c++17",
    "-lineinfo",
    "--expt-relaxed-constexpr",
    "-Xcompiler",
    "-fPIC",
    "-Xcompiler",
    "-fvisibility=hidden",
]


def sources() -> list[Path]:
    return sorted(CSRC.glob("*.cu"))


def _deps() -> list[Path]:
    return sources() + sorted(CSRC.glob("*.cuh")) + sorted(INCLUDE.glob("*.h"))


def _stale(target: Path, deps: list[Path]) -> bool:
    return not target.exists() or any(p.stat().st_mtime > target.stat().st_mtime for p in deps)


def needs_build() -> bool:
    return _stale(LIB_PATH, _deps()) or _stale(binding_path(), _binding_deps())


def binding_path() -> Path:
    """Where the binding for this Python and the installed torch is."""
    return LIB_DIR / f"_sa_paged-{sysconfig.get_config_var('SOABI')}-torch{importlib.metadata.version('torch')}.so"


def _binding_deps() -> list[Path]:
    return [BINDING_SRC, *sorted(INCLUDE.glob("*.h"))]


def build_binding(verbose: bool = False) -> Path:
    """Compile ``csrc/paged_binding.cpp`` against the installed torch (not imported)."""
    spec = importlib.util.find_spec("torch")
    if spec is None or spec.origin is None:
        raise RuntimeError("torch not found; the paged-cache binding cannot be built")
    torch = Path(spec.origin).parent
    cuda = Path(nvcc_path()).resolve().parent.parent
    path = binding_path()
    tmp = path.with_suffix(".so.tmp")
    cmd = [os.environ.get("CXX", "g++"), "-O2", "-std=c++17", "-fPIC", "-shared", "-fvisibility=hidden",
           "-D_GLIBCXX_USE_CXX11_ABI=1", "-I", sysconfig.get_paths()["include"], "-isystem", str(torch / "include"),
           "-isystem", str(torch / "include/torch/csrc/api/include"), "-isystem", str(cuda / "include"),
           str(BINDING_SRC), "-o", str(tmp), "-L", str(torch / "lib"), "-lc10", "-lc10_cuda", "-ltorch_cpu",
           "-ltorch_python"]
    if verbose:
        print(" ".join(cmd))
    subprocess.run(cmd, check=True)
    os.replace(tmp, path)
    return path


def nvcc_path() -> str:
    cand = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    if not Path(cand).exists():
        raise RuntimeError("nvcc not found; the sm_100a library cannot be built")
    return cand


def build(force: bool = False, verbose: bool = False, extra_flags: list[str] | None = None) -> Path:
    """Compile every ``csrc/*.cu`` into ``_lib/libsa_b200.so``, then the binding
    (each skipped when up to date)."""
    LIB_DIR.mkdir(exist_ok=True)
    if force or _stale(LIB_PATH, _deps()):
        build_library(verbose, extra_flags)
    if force or _stale(binding_path(), _binding_deps()):
        build_binding(verbose)
    return LIB_PATH


def build_library(verbose: bool = False, extra_flags: list[str] | None = None) -> Path:
    """Compile and link ``_lib/libsa_b200.so``."""
    nvcc = nvcc_path()
    objs = []
    build_dir = LIB_DIR / "obj"
    build_dir.mkdir(exist_ok=True)
    flags = ARCH_FLAGS + BASE_FLAGS + (extra_flags or [])
    if verbose:
        flags = flags + ["-Xptxas", "-v"]
    procs = []
    for src in sources():
        obj = build_dir / (src.stem + ".o")
        cmd = [nvcc, *flags, "-I", str(INCLUDE), "-c", str(src), "-o", str(obj)]
        procs.append((src, subprocess.Popen(cmd, stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True)))
        objs.append(obj)
    failed = []
    for src, p in procs:
        out, _ = p.communicate()
        if verbose or p.returncode != 0:
            sys.stderr.write(out)
        if p.returncode != 0:
            failed.append(src.name)
    if failed:
        raise RuntimeError(f"nvcc failed for {failed}")
    tmp = LIB_PATH.with_suffix(".so.tmp")
    link = [nvcc, *ARCH_FLAGS, "-shared", "-o", str(tmp), *map(str, objs)]
    subprocess.run(link, check=True)
    os.replace(tmp, LIB_PATH)
    return LIB_PATH


if __name__ == "__main__":
    force = "--force" in sys.argv
    verbose = "-v" in sys.argv or "--verbose" in sys.argv
    print(build(force=force, verbose=verbose))
