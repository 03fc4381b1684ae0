"""Build the native library ``libtidegs_amd.so`` from ``csrc/*.hip`` with hipcc, and the
Python modules ``_tensor_lists.so`` and ``_group_norm_node.so`` from ``csrc/*.cpp`` with g++.

Every translation unit of the library is compiled for gfx950 only, in parallel, and
linked into one shared object that exposes the C ABI declared in
``include/tidegs_amd.h``.  The library links only the HIP runtime: no torch
types cross the boundary.  The modules are host code alone: one reads lists of torch's
tensors into the rows of pointers that the library takes, one is a node of torch's
autograd graph that calls the library.
"""
from __future__ import annotations

import concurrent.futures as cf
import importlib.util
import os
import shutil
import subprocess
import sys
import sysconfig
from pathlib import Path

PKG_DIR = Path(__file__).resolve().parent
CSRC = PKG_DIR / "csrc"
OBJ_DIR = PKG_DIR / "_build"
LIB_PATH = PKG_DIR / "libtidegs_amd.so"
# Python modules of host code that knows torch's types: what each links beside torch's core
MODULES = {"tensor_lists": [], "group_norm_node": ["-lc10_hip"]}
ARCH = "gfx950"

HIPCC_FLAGS = [
    "-O3",
    "-std=c++17",
    f"--offload-arch={ARCH}",
    "-fPIC",
    "-munsafe-fp-atomics",
    # Packed-FP32 instruction forms stay disabled for every device pass.
    "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
    "-Wno-unused-result",
]


def _hipcc() -> str:
    for cand in (os.environ.get("HIPCC"), "/opt/rocm/bin/hipcc", shutil.which("hipcc")):
        if cand and Path(cand).exists():
            return cand
    raise RuntimeError("hipcc not found; the TideGS MI355X kernels need ROCm's hipcc")


def _compile(src: Path, hipcc: str) -> Path:
    obj = OBJ_DIR / (src.stem + ".o")
    cmd = [hipcc, *HIPCC_FLAGS, "-I", str(CSRC), "-c", str(src), "-o", str(obj)]
    proc = subprocess.run(cmd, capture_output=True, text=True)
    if proc.returncode != 0:
        raise RuntimeError(f"hipcc failed for {src.name}:\n{proc.stdout}\n{proc.stderr}")
    return obj


def _build_module(name: str) -> None:
    torch_dir = Path(importlib.util.find_spec("torch").origin).parent
    include, lib = torch_dir / "include", torch_dir / "lib"
    path = PKG_DIR / f"_{name}.so"
    tmp = path.with_suffix(".so.tmp")
    cmd = [shutil.which("g++") or "g++", "-O2", "-std=c++17", "-shared", "-fPIC", "-w",
           "-D__HIP_PLATFORM_AMD__", "-I", str(Path(_hipcc()).parents[1] / "include"),
           "-I", str(include), "-I", str(include / "torch" / "csrc" / "api" / "include"),
           "-I", sysconfig.get_paths()["include"], str(CSRC / f"{name}.cpp"), "-o", str(tmp),
           f"-L{lib}", f"-Wl,-rpath,{lib}", "-ltorch_python", "-ltorch_cpu", "-lc10",
           *MODULES[name]]
    proc = subprocess.run(cmd, capture_output=True, text=True)
    if proc.returncode != 0:
        raise RuntimeError(f"g++ failed for {name}.cpp:\n{proc.stdout}\n{proc.stderr}")
    os.replace(tmp, path)


def build(verbose: bool = False, jobs: int | None = None) -> Path:
    """Compile every HIP source and link ``libtidegs_amd.so``, and the modules; returns the
    library's path."""
    hipcc = _hipcc()
    OBJ_DIR.mkdir(exist_ok=True)
    sources = sorted(CSRC.glob("*.hip"))
    if not sources:
        raise RuntimeError(f"no HIP sources under {CSRC}")
    jobs = jobs or min(len(sources), max(1, min(8, os.cpu_count() or 1)))
    with cf.ThreadPoolExecutor(max_workers=jobs) as ex:
        modules = [ex.submit(_build_module, name) for name in MODULES]
        objs = list(ex.map(lambda s: _compile(s, hipcc), sources))
        for module in modules:
            module.result()
    tmp = LIB_PATH.with_suffix(".so.tmp")
    cmd = [hipcc, f"--offload-arch={ARCH}", "-shared", "-fPIC", *map(str, objs), "-o", str(tmp)]
    proc = subprocess.run(cmd, capture_output=True, text=True)
    if proc.returncode != 0:
        raise RuntimeError(f"link failed:\n{proc.stdout}\n{proc.stderr}")
    os.replace(tmp, LIB_PATH)
    if verbose:
        print(f"[tidegs_amd.build] {len(sources)} sources -> {LIB_PATH}")
    return LIB_PATH


if __name__ == "__main__":
    build(verbose=True)
    sys.exit(0)
