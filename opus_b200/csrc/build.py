"""Build libopus_b200.so in-tree with nvcc for sm_100a.

Usage: python -m opus_b200.csrc.build [--verbose]

Each .cu file is compiled to an object under opus_b200/_build/ (in parallel,
skipped when up to date) and linked into opus_b200/libopus_b200.so with the
CUDA runtime linked statically, so the library has no dependency on the
Python environment.  tensor_list.cpp becomes the extension module
opus_b200/_tensor_list.<this Python's tag>.so, against this Python's and
torch's headers; the library is built without it where it cannot be (no torch,
Python headers or C++ compiler), with a warning.
"""
from __future__ import annotations

import argparse
import concurrent.futures as cf
import importlib.util
import os
import shutil
import subprocess
import sys
import sysconfig
import warnings
from pathlib import Path

CSRC = Path(__file__).resolve().parent
PKG = CSRC.parent
ROOT = PKG.parent
BUILD = PKG / "_build"
LIB = PKG / "libopus_b200.so"
MODULE = PKG / ("_tensor_list" + sysconfig.get_config_var("EXT_SUFFIX"))

ARCH_FLAGS = ["-gencode", "arch=compute_100a,code=sm_100a"]
NVCC_FLAGS = ARCH_FLAGS + [
    "-O3",
    "-lineinfo",
    "-std=c++17",
    "--expt-relaxed-constexpr",
    "-Xcompiler", "-fPIC",
    "-Xcompiler", "-fvisibility=hidden",
    f"-I{ROOT / 'include'}",
]


def nvcc() -> str:
    for cand in (os.environ.get("NVCC"), shutil.which("nvcc"), "/usr/local/cuda/bin/nvcc"):
        if cand and Path(cand).exists():
            return cand
    raise RuntimeError("nvcc not found: cannot build libopus_b200.so")


def sources() -> list[Path]:
    return sorted(CSRC.glob("*.cu"))


def headers() -> list[Path]:
    return sorted(CSRC.glob("*.cuh")) + sorted(CSRC.glob("*.h")) + sorted((ROOT / "include").glob("*.h"))


def _stale(obj: Path, src: Path, deps: list[Path]) -> bool:
    if not obj.exists():
        return True
    t = obj.stat().st_mtime
    return any(p.stat().st_mtime > t for p in [src, *deps])


def _compile(src: Path, verbose: bool, extra: list[str]) -> Path:
    obj = BUILD / (src.stem + ".o")
    cmd = [nvcc(), *NVCC_FLAGS, *extra, "-c", str(src), "-o", str(obj)]
    if verbose:
        print(" ".join(cmd), flush=True)
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError(f"nvcc failed on {src.name}:\n{res.stdout}\n{res.stderr}")
    if verbose and (res.stdout or res.stderr):
        print(res.stdout + res.stderr, flush=True)
    return obj


def build_module(verbose: bool = False, force: bool = False) -> Path:
    """The extension module that walks lists of torch tensors; RuntimeError where it cannot be built."""
    src = CSRC / "tensor_list.cpp"
    spec = importlib.util.find_spec("torch")
    if spec is None or spec.origin is None:
        raise RuntimeError(f"torch not found: cannot build {MODULE.name}")
    torch_dir = Path(spec.origin).resolve().parent
    cuda_include = Path(nvcc()).resolve().parent.parent / "include"
    if not force and not _stale(MODULE, src, [ROOT / "include" / "opus_b200.h", torch_dir / "version.py"]):
        return MODULE
    tmp = MODULE.with_suffix(".so.tmp")
    cmd = [os.environ.get("CXX") or shutil.which("g++") or "c++", "-O2", "-std=c++17", "-shared", "-fPIC",
           "-fvisibility=hidden", f"-I{sysconfig.get_paths()['include']}", "-isystem", str(torch_dir / "include"),
           "-isystem", str(torch_dir / "include" / "torch" / "csrc" / "api" / "include"), "-isystem", str(cuda_include),
           str(src), f"-L{torch_dir / 'lib'}", "-ltorch_python", "-ltorch_cpu", "-lc10", "-o", str(tmp)]
    if verbose:
        print(" ".join(cmd), flush=True)
    try:
        res = subprocess.run(cmd, capture_output=True, text=True)
    except OSError as e:
        raise RuntimeError(f"no C++ compiler for {src.name}: {e}") from e
    if res.returncode != 0:
        raise RuntimeError(f"c++ failed on {src.name}:\n{res.stdout}\n{res.stderr}")
    os.replace(tmp, MODULE)
    return MODULE


def build(verbose: bool = False, force: bool = False, extra: list[str] | None = None) -> Path:
    extra = list(extra or [])
    BUILD.mkdir(parents=True, exist_ok=True)
    deps = headers()
    srcs = sources()
    todo = [s for s in srcs if force or extra or _stale(BUILD / (s.stem + ".o"), s, deps)]
    with cf.ThreadPoolExecutor(max_workers=8) as ex:
        module = ex.submit(build_module, verbose, force)
        list(ex.map(lambda s: _compile(s, verbose, extra), todo))
    objs = [BUILD / (s.stem + ".o") for s in srcs]
    if todo or not LIB.exists() or any(o.stat().st_mtime > LIB.stat().st_mtime for o in objs):
        tmp = LIB.with_suffix(".so.tmp")
        cmd = [nvcc(), *ARCH_FLAGS, "-shared", "-cudart", "static", "-o", str(tmp), *map(str, objs)]
        if verbose:
            print(" ".join(cmd), flush=True)
        res = subprocess.run(cmd, capture_output=True, text=True)
        if res.returncode != 0:
            raise RuntimeError(f"link failed:\n{res.stdout}\n{res.stderr}")
        os.replace(tmp, LIB)
    if module.exception() is not None:
        if not isinstance(module.exception(), RuntimeError):
            raise module.exception()
        warnings.warn(f"{LIB.name} is built, {MODULE.name} could not be (operators on lists of tensors need it): "
                      f"{module.exception()}", RuntimeWarning, stacklevel=2)
    return LIB


def main(argv: list[str] | None = None) -> int:
    ap = argparse.ArgumentParser()
    ap.add_argument("--verbose", action="store_true")
    ap.add_argument("--force", action="store_true")
    ap.add_argument("--ptxas-info", action="store_true", help="print registers/spills per kernel")
    args = ap.parse_args(argv)
    extra = ["-Xptxas", "-v"] if args.ptxas_info else []
    lib = build(verbose=args.verbose or args.ptxas_info, force=args.force, extra=extra)
    print(lib)
    return 0


if __name__ == "__main__":
    sys.exit(main())
