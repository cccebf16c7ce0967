"""Build recipe for the native library: nvcc, sm_100a, in-tree.

    python -m blackwell_b200.build        # -> blackwell_b200/libbw_attn.so

It also links the C++ harness ``bw_harness`` (harness/bw_harness.cpp) and the
torch front end of the cache calls ``_front.so`` (front/front.cpp, a CPython
module; left out where torch's or Python's headers are missing) against the
library.  Every .cu under csrc/ is compiled with
``-gencode arch=compute_100a,code=sm_100a -lineinfo -O3`` and linked into one
shared library with the CUDA runtime linked statically (no torch types cross
the boundary; the library only depends on the driver at run time).
"""
from __future__ import annotations

import os
import shutil
import subprocess
import sys
import sysconfig
from concurrent.futures import ThreadPoolExecutor
from pathlib import Path

HERE = Path(__file__).resolve().parent
CSRC = HERE / "csrc"
OUT = HERE / "libbw_attn.so"
HARNESS = HERE / "bw_harness"
HARNESS_SRC = HERE / "harness" / "bw_harness.cpp"
FRONT = HERE / "_front.so"
FRONT_SRC = HERE / "front" / "front.cpp"
BUILD = HERE / "_build"
NVCC = os.environ.get("NVCC", "/usr/local/cuda/bin/nvcc")
FLAGS = ["-gencode", "arch=compute_100a,code=sm_100a", "-lineinfo", "-O3", "-std=c++17",
         "-Xcompiler", "-fPIC", "-Xcompiler", "-fvisibility=hidden", "--expt-relaxed-constexpr"]


def _sources():
    return sorted(CSRC.glob("*.cu"))


def _deps():
    return sorted(CSRC.glob("*.cu*")) + sorted(CSRC.glob("*.h")) + sorted((HERE.parent / "include").glob("*.h"))


def up_to_date() -> bool:
    built = [OUT, HARNESS] if front_lacks() else [OUT, HARNESS, FRONT]
    if not all(p.exists() for p in built):
        return False
    if FRONT in built and not front_fits():
        return False
    t = min(p.stat().st_mtime for p in built)
    return all(p.stat().st_mtime <= t for p in _deps() + [HARNESS_SRC, FRONT_SRC])


def build(force: bool = False, verbose: bool = False) -> Path:
    if not force and up_to_date():
        return OUT
    BUILD.mkdir(exist_ok=True)

    def compile_one(src: Path) -> Path:
        obj = BUILD / (src.stem + ".o")
        cmd = [NVCC, *FLAGS, "-c", str(src), "-o", str(obj)]
        if verbose:
            print(" ".join(cmd))
        subprocess.run(cmd, check=True)
        return obj

    with ThreadPoolExecutor(max_workers=os.cpu_count() or 4) as ex:
        objs = list(ex.map(compile_one, _sources()))
    tmp = OUT.with_suffix(".so.tmp")
    cmd = [NVCC, "-shared", "-gencode", "arch=compute_100a,code=sm_100a", "-o", str(tmp), *map(str, objs)]
    subprocess.run(cmd, check=True)
    os.replace(tmp, OUT)
    build_harness(verbose)
    build_front(verbose)
    return OUT


def front_lacks():
    """What the torch front end cannot be built without and is not here, or None."""
    try:
        import torch
    except ImportError:
        return "torch"
    for what, there in (("g++", shutil.which("g++")),
                        ("Python.h", (Path(sysconfig.get_paths()["include"]) / "Python.h").exists()),
                        ("torch's headers", (Path(torch.__file__).resolve().parent / "include" / "ATen").is_dir())):
        if not there:
            return what
    return None


def front_fits() -> bool:
    """Whether the torch front end was built with this torch (its version stands in the file)."""
    import torch
    return torch.__version__.encode() + b"\0" in FRONT.read_bytes()


def build_front(verbose: bool = False):
    """The torch front end: a CPython module over the C ABI, linked to the library.
    Where the box has no headers for it, it is left out (the calls of cache.py say
    so when they are used); the library and the harness do not need it."""
    lacks = front_lacks()
    if lacks:
        print(f"{FRONT.name} is not built: {lacks} not found", file=sys.stderr)
        return None
    import torch
    cuda = Path(shutil.which(NVCC) or NVCC).resolve().parent.parent
    root = Path(torch.__file__).resolve().parent
    tmp = FRONT.with_suffix(".so.tmp")
    cmd = ["g++", "-O2", "-std=c++17", "-shared", "-fPIC", "-fvisibility=hidden",
           f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}", f'-DBW_FRONT_TORCH="{torch.__version__}"']
    for p in (root / "include", root / "include" / "torch" / "csrc" / "api" / "include",
              cuda / "include", sysconfig.get_paths()["include"]):
        cmd += ["-isystem", str(p)]
    cmd += [str(FRONT_SRC), "-o", str(tmp), "-L", str(HERE), "-lbw_attn", "-Wl,-rpath,$ORIGIN",
            "-L", str(root / "lib"), "-ltorch_python", "-ltorch_cpu", "-lc10", "-lc10_cuda"]
    if verbose:
        print(" ".join(cmd))
    subprocess.run(cmd, check=True)
    os.replace(tmp, FRONT)
    return FRONT


def build_harness(verbose: bool = False) -> Path:
    """The C++ harness (reference-style main over the C ABI), linked to the library."""
    cmd = [NVCC, "-gencode", "arch=compute_100a,code=sm_100a", "-O3", "-std=c++17", "-I", str(HERE.parent / "include"),
           str(HARNESS_SRC), "-o", str(HARNESS),
           "-L", str(HERE), "-lbw_attn", "-Xlinker", "-rpath,$ORIGIN"]
    if verbose:
        print(" ".join(cmd))
    subprocess.run(cmd, check=True)
    return HARNESS


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose=True))
