"""Build the dot_b200 C-ABI library for sm_100a with nvcc (in-tree).

``python dot_b200/build.py`` compiles every ``csrc/*.cu`` (in parallel, one
object per source under ``dot_b200/_lib/obj``) and links them into
``dot_b200/_lib/libdot_b200.so``, with
``-gencode arch=compute_100a,code=sm_100a -lineinfo -O3``.  The CUDA runtime is
linked statically so the library carries no dependency beyond the driver
(NCCL, used only by the row-sharded solver, is loaded at run time).
``csrc/torch_features.cpp``, the torch binding of the feature operators, is
compiled with the host compiler against the installed torch and linked to that
library (``_lib/_torch_features.so``).  Each is skipped when it is newer than
its sources, the binding if it was also built for the torch and Python that run.
"""

from __future__ import annotations

import glob
import os
from concurrent.futures import ThreadPoolExecutor
import shutil
import subprocess
import sys

HERE = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(HERE)
LIB_DIR = os.path.join(HERE, "_lib")
LIB = os.path.join(LIB_DIR, "libdot_b200.so")
BINDING = os.path.join(LIB_DIR, "_torch_features.so")
BINDING_STAMP = os.path.join(LIB_DIR, "_torch_features.built_for")   # the torch and Python it was compiled against
BINDING_SRC = os.path.join(HERE, "csrc", "torch_features.cpp")
ARCH = "-gencode=arch=compute_100a,code=sm_100a"


def _nvcc() -> str:
    for cand in (os.environ.get("NVCC"), shutil.which("nvcc"), "/usr/local/cuda/bin/nvcc"):
        if cand and os.path.exists(cand):
            return cand
    raise RuntimeError("nvcc not found; set NVCC or put the CUDA toolkit on PATH")


def sources() -> list[str]:
    return sorted(glob.glob(os.path.join(HERE, "csrc", "*.cu")))


def _stale() -> bool:
    if not os.path.exists(LIB):
        return True
    t = os.path.getmtime(LIB)
    deps = sources() + glob.glob(os.path.join(HERE, "csrc", "*.h")) + glob.glob(
        os.path.join(HERE, "csrc", "*.cuh")) + glob.glob(os.path.join(ROOT, "include", "*.h"))
    return any(os.path.getmtime(d) > t for d in deps)


def _binding_stale(built_for: str) -> bool:
    if not os.path.exists(BINDING) or not os.path.exists(BINDING_STAMP):
        return True
    with open(BINDING_STAMP) as f:
        if f.read() != built_for:
            return True
    deps = [BINDING_SRC, os.path.join(ROOT, "include", "dot_b200.h")]
    return any(os.path.getmtime(d) > os.path.getmtime(BINDING) for d in deps)


def build_binding(force: bool = False, verbose: bool = False) -> str:
    """The torch binding: host code only, linked to libdot_b200.so beside it."""
    import sysconfig

    import torch

    built_for = f"torch {torch.__version__}, {sysconfig.get_config_var('SOABI')}"
    if not force and not _binding_stale(built_for):
        return BINDING
    from torch.utils import cpp_extension

    cuda = os.path.dirname(os.path.dirname(os.path.realpath(_nvcc())))
    tmp = BINDING + ".tmp"
    # the system compiler, whose C++ library the process runs on (not $CXX, which may bring another)
    cmd = ["/usr/bin/g++" if os.path.exists("/usr/bin/g++") else "g++", "-O2", "-std=c++17", "-fPIC", "-shared", "-fvisibility=hidden", "-w",
           "-DTORCH_EXTENSION_NAME=_torch_features",
           f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}"]
    cmd += ["-I" + p for p in cpp_extension.include_paths() + [sysconfig.get_paths()["include"],
                                                                os.path.join(cuda, "include")]]
    cmd += [BINDING_SRC, "-o", tmp, "-L" + LIB_DIR, "-l:libdot_b200.so", "-Wl,-rpath,$ORIGIN"]
    cmd += ["-L" + p for p in cpp_extension.library_paths()]
    cmd += ["-ltorch_python", "-ltorch", "-ltorch_cpu", "-lc10_cuda", "-lc10"]
    if verbose:
        print(" ".join(cmd), file=sys.stderr)
    subprocess.run(cmd, check=True)
    os.replace(tmp, BINDING)
    with open(BINDING_STAMP, "w") as f:
        f.write(built_for)
    return BINDING


def build(force: bool = False, verbose: bool = False) -> str:
    if force or _stale():
        _build_library(verbose)
    build_binding(force, verbose)
    return LIB


def _build_library(verbose: bool) -> None:
    obj_dir = os.path.join(LIB_DIR, "obj")
    os.makedirs(obj_dir, exist_ok=True)
    flags = [ARCH, "-lineinfo", "-O3", "-std=c++17", "-Xcompiler", "-fPIC", "-Xcompiler", "-fvisibility=hidden",
             "--expt-relaxed-constexpr", "-I" + os.path.join(ROOT, "include")]
    nvcc = _nvcc()

    def compile_one(src: str) -> str:
        obj = os.path.join(obj_dir, os.path.splitext(os.path.basename(src))[0] + ".o")
        cmd = [nvcc] + flags + ["-c", src, "-o", obj]
        if verbose:
            print(" ".join(cmd), file=sys.stderr)
        subprocess.run(cmd, check=True)
        return obj

    with ThreadPoolExecutor(max_workers=max(1, min(len(sources()), os.cpu_count() or 1))) as ex:
        objs = list(ex.map(compile_one, sources()))
    tmp = LIB + ".tmp"
    cmd = [nvcc, ARCH, "-shared", "-cudart", "static", "-o", tmp] + objs + ["-ldl"]
    if verbose:
        print(" ".join(cmd), file=sys.stderr)
    subprocess.run(cmd, check=True)
    os.replace(tmp, LIB)


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose=True))
