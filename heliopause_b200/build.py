"""Builds libheliocuda.so in-tree with nvcc for sm_100a (no GPU needed), and
the host module _host.so beside it with g++ (csrc/hc_host.cpp, on torch's headers).

    python -m heliopause_b200.build          # incremental
    python -m heliopause_b200.build --force  # rebuild everything
"""
from __future__ import annotations

import argparse
import importlib.util
import os
import shutil
import subprocess
import sys
import sysconfig
from concurrent.futures import ThreadPoolExecutor
from pathlib import Path

from . import _lib

PKG = Path(__file__).resolve().parent
CSRC = PKG / "csrc"
OBJ = PKG / "_build"
LIB = PKG / "libheliocuda.so"
HOST_SRC = CSRC / "hc_host.cpp"
HOST_LIB = PKG / "_host.so"
NVCC = os.environ.get("NVCC", "/usr/local/cuda/bin/nvcc")
CXX = os.environ.get("CXX", "g++")
ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]
FLAGS = ["-O3", "-lineinfo", "-std=c++17", "-Xcompiler", "-fPIC", "--expt-relaxed-constexpr",
         "-Xptxas", "-warn-spills"]


def _sources() -> list[Path]:
    return sorted(CSRC.glob("*.cu"))


def _headers() -> list[Path]:
    return sorted(CSRC.glob("*.cuh")) + sorted((PKG.parent / "include").glob("*.h"))


def _build_host(force: bool) -> None:
    hdr = PKG.parent / "include" / "heliocuda.h"
    stamp = OBJ / "_host.built_for"
    if not force and HOST_LIB.exists() and HOST_LIB.stat().st_mtime > max(HOST_SRC.stat().st_mtime, hdr.stat().st_mtime) \
            and stamp.exists() and stamp.read_text() == _lib.host_built_for():
        return
    torch = Path(importlib.util.find_spec("torch").origin).parent
    inc = [torch / "include", torch / "include/torch/csrc/api/include", sysconfig.get_paths()["include"],
           Path(shutil.which(NVCC) or NVCC).resolve().parents[1] / "include", hdr.parent]
    cmd = [CXX, "-O2", "-std=c++17", "-fPIC", "-shared", f'-DHC_BUILT_FOR="{_lib.host_built_for()}"',
           *(f"-I{i}" for i in inc), str(HOST_SRC), "-o", str(HOST_LIB), f"-L{torch / 'lib'}", "-ltorch_python", "-ltorch",
           "-ltorch_cpu", "-lc10", "-lc10_cuda"]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        sys.stderr.write(r.stdout + r.stderr)
        raise RuntimeError(f"{CXX} failed on {HOST_SRC.name}")
    stamp.write_text(_lib.host_built_for())


def build(force: bool = False, verbose: bool = False, extra: list[str] | None = None) -> Path:
    OBJ.mkdir(exist_ok=True)
    hdr_mtime = max((h.stat().st_mtime for h in _headers()), default=0.0)
    jobs = []
    for src in _sources():
        obj = OBJ / (src.stem + ".o")
        if force or not obj.exists() or obj.stat().st_mtime < max(src.stat().st_mtime, hdr_mtime):
            cmd = [NVCC, *ARCH, *FLAGS, *(extra or []), "-c", str(src), "-o", str(obj)]
            jobs.append((src, cmd))

    def run(job):
        src, cmd = job
        r = subprocess.run(cmd, capture_output=True, text=True)
        return src, r

    with ThreadPoolExecutor(max_workers=min(8, os.cpu_count() or 1)) as ex:
        for src, r in ex.map(run, jobs):
            if verbose or r.returncode != 0:
                sys.stderr.write(r.stdout + r.stderr)
            if r.returncode != 0:
                raise RuntimeError(f"nvcc failed on {src.name}")
    objs = [OBJ / (s.stem + ".o") for s in _sources()]
    if force or jobs or not LIB.exists():
        cmd = [NVCC, *ARCH, "-shared", "-o", str(LIB), *map(str, objs), "-lcuda"]
        r = subprocess.run(cmd, capture_output=True, text=True)
        if r.returncode != 0:
            sys.stderr.write(r.stdout + r.stderr)
            raise RuntimeError("link failed")
    _build_host(force)
    return LIB


if __name__ == "__main__":
    ap = argparse.ArgumentParser()
    ap.add_argument("--force", action="store_true")
    ap.add_argument("-v", "--verbose", action="store_true")
    a = ap.parse_args()
    print(build(force=a.force, verbose=a.verbose))
