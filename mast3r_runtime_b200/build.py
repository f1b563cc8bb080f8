"""Build libm3r_cuda.so (sm_100a) in-tree with nvcc, and the torch side of ops.py with g++.

    python -m mast3r_runtime_b200.build          # or: python mast3r_runtime_b200/build.py

Objects go to mast3r_runtime_b200/_build/ (rebuilt when a source or header is newer);
the shared libraries are written next to this file so that they travel with the tree.
_torch_ops.so (binding/torch_ops.cpp, the tensors of mast3r_runtime_b200.ops) is built against the
torch of this interpreter, and left out where that is not there, has no CUDA or no headers: nothing else
in the package needs it.
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

HERE = Path(__file__).resolve().parent
CSRC = HERE / "csrc"
BUILD = HERE / "_build"
LIB = HERE / "libm3r_cuda.so"
INCLUDE = HERE.parent / "include"
BINDING = HERE / "binding" / "torch_ops.cpp"
TORCH_LIB = HERE / "_torch_ops.so"
TORCH_STAMP = HERE / "_torch_ops.stamp"  # what it was built for; travels with it

ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]
NVCC_FLAGS = ["-std=c++17", "-O3", "-lineinfo", "-Xcompiler", "-fPIC", "-Xcompiler", "-fvisibility=hidden",
              "-Xcompiler", "-Wno-attributes", "--expt-relaxed-constexpr"]


def nvcc() -> str:
    for cand in (os.environ.get("NVCC"), shutil.which("nvcc"), "/usr/local/cuda/bin/nvcc"):
        if cand and Path(cand).exists():
            return cand
    raise RuntimeError("nvcc not found")


def _sources():
    return sorted(list(CSRC.glob("*.cu")) + list(CSRC.glob("*.cpp")))


def _headers_mtime() -> float:
    hs = list(CSRC.glob("*.h")) + list(CSRC.glob("*.cuh")) + list(INCLUDE.glob("*.h"))
    return max((h.stat().st_mtime for h in hs), default=0.0)


def _compile(src: Path, hmt: float) -> Path:
    obj = BUILD / (src.name + ".o")
    if obj.exists() and obj.stat().st_mtime >= max(src.stat().st_mtime, hmt):
        return obj
    cmd = [nvcc(), *ARCH, *NVCC_FLAGS, "-I", str(INCLUDE), "-c", str(src), "-o", str(obj)]
    if src.suffix == ".cpp":
        cmd = [nvcc(), *NVCC_FLAGS, "-x", "cu", *ARCH, "-I", str(INCLUDE), "-c", str(src), "-o", str(obj)]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"nvcc failed for {src.name}:\n{r.stdout}\n{r.stderr}")
    return obj


def build(verbose: bool = False) -> Path:
    BUILD.mkdir(exist_ok=True)
    hmt = _headers_mtime()
    srcs = _sources()
    with cf.ThreadPoolExecutor(max_workers=min(8, len(srcs))) as ex:
        objs = list(ex.map(lambda s: _compile(s, hmt), srcs))
    newest = max(o.stat().st_mtime for o in objs)
    if not LIB.exists() or LIB.stat().st_mtime < newest:
        # static cudart: the library does not depend on whichever libcudart a host process loaded first
        cmd = [nvcc(), *ARCH, "-shared", "-cudart", "static", "-o", str(LIB), *map(str, objs), "-lpthread", "-lrt", "-ldl"]
        r = subprocess.run(cmd, capture_output=True, text=True)
        if r.returncode != 0:
            raise RuntimeError(f"link failed:\n{r.stdout}\n{r.stderr}")
    if verbose:
        print(f"built {LIB}")
    binding = build_torch_ops()
    if verbose and binding:
        print(f"built {binding}")
    return LIB


def _missing_for_torch_ops(torch: Path | None) -> str | None:
    """What the binding needs and this interpreter does not have."""
    if torch is None:
        return "no torch"
    for lib in ("libtorch_python.so", "libtorch_cuda.so", "libc10_cuda.so"):
        if not (torch / "lib" / lib).exists():
            return f"torch without {lib}"
    if not (torch / "include" / "ATen" / "ATen.h").exists():
        return "torch without headers"
    if not (Path(sysconfig.get_paths()["include"]) / "Python.h").exists():
        return "no Python headers"
    return None


def build_torch_ops() -> Path | None:
    """_torch_ops.so, rebuilt when its source, the C header, torch's or Python's version changed; None
    where it is left out."""
    spec = importlib.util.find_spec("torch")
    root = Path(spec.origin).parent if spec is not None and spec.origin else None
    missing = _missing_for_torch_ops(root)
    if missing:
        print(f"{missing}: mast3r_runtime_b200.ops is not built", file=sys.stderr)
        TORCH_LIB.unlink(missing_ok=True)
        return None
    version = (root / "version.py").read_text() + f"python {sysconfig.get_config_var('SOABI')}\n"
    newest = max(BINDING.stat().st_mtime, (INCLUDE / "m3r_cuda.h").stat().st_mtime)
    if (TORCH_LIB.exists() and TORCH_LIB.stat().st_mtime >= newest and TORCH_STAMP.exists()
            and TORCH_STAMP.read_text() == version):
        return TORCH_LIB
    cuda = Path(nvcc()).resolve().parent.parent / "include"
    tmp = BUILD / TORCH_LIB.name
    cmd = [os.environ.get("CXX", "g++"), "-std=c++17", "-O2", "-fPIC", "-shared", "-fvisibility=hidden",
           "-I", sysconfig.get_paths()["include"], "-isystem", str(root / "include"),
           "-isystem", str(root / "include" / "torch" / "csrc" / "api" / "include"), "-isystem", str(cuda),
           str(BINDING), "-o", str(tmp), "-L", str(HERE), f"-l:{LIB.name}", "-L", str(root / "lib"),
           "-ltorch_python", "-ltorch", "-ltorch_cpu", "-ltorch_cuda", "-lc10", "-lc10_cuda", "-Wl,-rpath,$ORIGIN"]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"{cmd[0]} failed for {BINDING.name}:\n{r.stdout}\n{r.stderr}")
    os.replace(tmp, TORCH_LIB)
    TORCH_STAMP.write_text(version)
    return TORCH_LIB


if __name__ == "__main__":
    build(verbose=True)
    sys.exit(0)
