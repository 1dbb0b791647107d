"""Builds the firepit_b200 CUDA library in-tree: firepit_b200/libfirepit_b200.so,
and firepit_b200/_calls.so, which makes the paged cache's calls on torch's tensors
(csrc/calls.cpp).

Every translation unit is compiled for sm_100a only
(``-gencode arch=compute_100a,code=sm_100a``), objects go to
``firepit_b200/_build/`` and the shared library links the CUDA runtime
statically, so the .so that travels with the source tree is self-contained.
Rebuilds only what changed (sources or any header).
"""
from __future__ import annotations

import concurrent.futures as cf
import importlib.util
import os
import runpy
import shutil
import subprocess
import sys
import sysconfig
import warnings
from pathlib import Path

PKG = Path(__file__).resolve().parent
CSRC = PKG / "csrc"
BUILD = PKG / "_build"
LIB = PKG / "libfirepit_b200.so"
CALLS = PKG / "_calls.so"
INCLUDE = PKG.parent / "include"

ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]
NVCC_FLAGS = ["-O3", "-lineinfo", "-std=c++17", "-Xcompiler", "-fPIC", "--expt-relaxed-constexpr",
              "-Xptxas", "-warn-spills"] + ARCH


def nvcc() -> str:
    for cand in (os.environ.get("NVCC"), shutil.which("nvcc"), "/usr/local/cuda/bin/nvcc"):
        if cand and Path(cand).exists():
            return cand
    raise RuntimeError("nvcc not found")


def _headers() -> list[Path]:
    return sorted(CSRC.glob("*.cuh")) + sorted(INCLUDE.glob("*.h"))


def _stale(src: Path, obj: Path, newest_header: float) -> bool:
    if not obj.exists():
        return True
    t = obj.stat().st_mtime
    return src.stat().st_mtime > t or newest_header > t


def _compile(src: Path, obj: Path, verbose: bool) -> tuple[Path, str]:
    cmd = [nvcc(), *NVCC_FLAGS, "-I", str(INCLUDE), "-c", str(src), "-o", str(obj)]
    if verbose:
        cmd += ["-Xptxas", "-v"]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"nvcc failed for {src.name}:\n{r.stdout}\n{r.stderr}")
    return src, r.stderr


def build(verbose: bool = False, force: bool = False) -> Path:
    BUILD.mkdir(exist_ok=True)
    sources = sorted(CSRC.glob("*.cu"))
    newest = max((h.stat().st_mtime for h in _headers()), default=0.0)
    jobs = []
    for src in sources:
        obj = BUILD / (src.stem + ".o")
        if force or verbose or _stale(src, obj, newest):
            jobs.append((src, obj))
    if jobs:
        with cf.ThreadPoolExecutor(max_workers=min(len(jobs), os.cpu_count() or 4)) as ex:
            for src, log in ex.map(lambda j: _compile(*j, verbose), jobs):
                if verbose and log:
                    print(f"== {src.name}\n{log}", file=sys.stderr)
    objs = [BUILD / (s.stem + ".o") for s in sources]
    if force or jobs or not LIB.exists() or any(o.stat().st_mtime > LIB.stat().st_mtime for o in objs):
        tmp = LIB.with_suffix(".so.tmp")
        cmd = [nvcc(), "-shared", *ARCH, "-o", str(tmp), *map(str, objs), "-cudart", "static"]
        r = subprocess.run(cmd, capture_output=True, text=True)
        if r.returncode != 0:
            raise RuntimeError(f"link failed:\n{r.stdout}\n{r.stderr}")
        os.replace(tmp, LIB)
    _build_calls(force)
    return LIB


def _build_calls(force: bool) -> None:
    """The module links torch and the library above (found beside it), for the torch
    and the Python that are here: it is made again for others.  It saves a call some
    microseconds and nothing else needs it, so what keeps it from being built is noted
    and an older one removed (the calls go by ctypes)."""
    spec = importlib.util.find_spec("torch")
    if spec is None or spec.origin is None:
        return
    src, torch, stamp = CSRC / "calls.cpp", Path(spec.origin).parent, BUILD / "calls.for"
    tmp = CALLS.with_suffix(".so.tmp")
    try:
        made_for = f"{runpy.run_path(str(torch / 'version.py'))['__version__']} {sys.implementation.cache_tag}"
        newest = max(p.stat().st_mtime for p in (src, INCLUDE / "firepit_b200.h"))
        if not force and CALLS.exists() and newest <= CALLS.stat().st_mtime and stamp.exists() and (
                stamp.read_text() == made_for):
            return
        cuda = Path(nvcc()).resolve().parent.parent
        cmd = ["g++", "-O2", "-std=c++17", "-fPIC", "-shared", "-fvisibility=hidden", f'-DFPB_CALLS_FOR="{made_for}"',
               *(f"-I{p}" for p in (INCLUDE, torch / "include", torch / "include/torch/csrc/api/include",
                                    sysconfig.get_paths()["include"], cuda / "include")),
               str(src), "-o", str(tmp), f"-L{PKG}", f"-l:{LIB.name}", f"-L{torch / 'lib'}", "-ltorch_python", "-ltorch",
               "-ltorch_cpu", "-lc10", "-lc10_cuda", "-Wl,-rpath,$ORIGIN"]
        r = subprocess.run(cmd, capture_output=True, text=True)
        if r.returncode != 0:
            raise RuntimeError(f"g++ failed for {src.name}:\n{r.stdout}\n{r.stderr}")
        os.replace(tmp, CALLS)
        stamp.write_text(made_for)
    except (OSError, RuntimeError, KeyError) as e:
        CALLS.unlink(missing_ok=True)
        warnings.warn(f"{CALLS.name} was not built, the paged cache's calls go by ctypes: {e}", stacklevel=2)


if __name__ == "__main__":
    build(verbose="-v" in sys.argv, force="-f" in sys.argv)
    print(LIB)
