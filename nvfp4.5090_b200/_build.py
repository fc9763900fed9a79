"""In-tree build of the CUDA library ``lib/libnvfp4b200.so`` (sm_100a only).

nvcc compiles each ``csrc/*.cu`` for ``-gencode arch=compute_100a,code=sm_100a``
into ``_build/`` and links one shared object with the CUDA runtime linked
statically, so the library depends only on the driver (libcuda) at run time
and can be loaded next to any PyTorch build.  ``build_binding`` compiles the
torch extension module on top of it (csrc/torch_binding.cpp, host code only)
against the installed PyTorch.
"""
from __future__ import annotations

import os
import shutil
import subprocess
import sys
from concurrent.futures import ThreadPoolExecutor

PKG_DIR = os.path.dirname(os.path.abspath(__file__))
REPO_DIR = os.path.dirname(PKG_DIR)
CSRC = os.path.join(PKG_DIR, "csrc")
BUILD_DIR = os.path.join(PKG_DIR, "_build")
LIB_DIR = os.path.join(PKG_DIR, "lib")
LIB_PATH = os.path.join(LIB_DIR, "libnvfp4b200.so")
BINDING_NAME = "_nvfp4b200_torch"
BINDING_PATH = os.path.join(LIB_DIR, BINDING_NAME + ".so")
BINDING_STAMP = os.path.join(LIB_DIR, BINDING_NAME + ".txt")   # what the module was compiled against
SOURCES = ["quant.cu", "gemm.cu", "train.cu", "noalloc.cu", "mx.cu", "mxlin.cu", "clip.cu", "norm.cu"]
HEADERS = [os.path.join(CSRC, "common.cuh"), os.path.join(CSRC, "vec.cuh"), os.path.join(CSRC, "bulk.cuh"), os.path.join(CSRC, "mx.cuh"),
           os.path.join(CSRC, "sched_slots.h"), os.path.join(CSRC, "row_stop.h"), os.path.join(REPO_DIR, "include", "nvfp4_b200.h")]
ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]
NVCC_FLAGS = ["-std=c++17", "-O3", "-lineinfo", "-Xcompiler", "-fPIC", "--expt-relaxed-constexpr"] + ARCH


def _nvcc() -> str:
    for cand in (os.environ.get("NVCC"), shutil.which("nvcc"), "/usr/local/cuda/bin/nvcc"):
        if cand and os.path.exists(cand):
            return cand
    raise RuntimeError("nvcc not found: the NVFP4 B200 library must be compiled with the CUDA toolkit")


def _stale(target: str, deps) -> bool:
    if not os.path.exists(target):
        return True
    t = os.path.getmtime(target)
    return any(os.path.getmtime(d) > t for d in deps)


def build(force: bool = False, verbose: bool = False) -> str:
    """Compile (if needed) and return the path of the shared library."""
    nvcc = _nvcc()
    os.makedirs(BUILD_DIR, exist_ok=True)
    os.makedirs(LIB_DIR, exist_ok=True)
    objs, todo = [], []
    for src in SOURCES:
        s = os.path.join(CSRC, src)
        o = os.path.join(BUILD_DIR, src.replace(".cu", ".o"))
        objs.append(o)
        if force or _stale(o, [s] + HEADERS):
            todo.append([nvcc] + NVCC_FLAGS + ["-c", s, "-o", o])
    if verbose:
        for cmd in todo:
            print(" ".join(cmd), file=sys.stderr)
    # side by side: norm.cu alone (360 kernels) takes two to three minutes.  (Not with nvcc's
    # --split-compile, half of that: the forward norm at 16384 x 8192 then took 210 us, 190 without.)
    with ThreadPoolExecutor(max_workers=os.cpu_count() or 1) as pool:
        for done in [pool.submit(subprocess.run, cmd, check=True) for cmd in todo]:
            done.result()
    if force or _stale(LIB_PATH, objs):
        tmp = LIB_PATH + ".tmp"
        cmd = [nvcc, "-shared"] + ARCH + ["-o", tmp] + objs
        if verbose:
            print(" ".join(cmd), file=sys.stderr)
        subprocess.run(cmd, check=True)
        os.replace(tmp, LIB_PATH)
    build_binding(force, verbose)
    return LIB_PATH


def binding_target() -> str:
    """The PyTorch and Python whose binary interfaces the torch extension module is made for."""
    import torch
    return f"torch {torch.__version__}, C++11 ABI {int(torch._C._GLIBCXX_USE_CXX11_ABI)}, {sys.implementation.cache_tag}"


def binding_built_for() -> str:
    """``binding_target()`` at the time the module was built; empty where nothing tells."""
    if not os.path.exists(BINDING_STAMP):
        return ""
    with open(BINDING_STAMP) as f:
        return f.read().strip()


def build_binding(force: bool = False, verbose: bool = False) -> str:
    """Compile (if needed: sources newer, or another PyTorch or Python) the
    torch extension module next to the library."""
    src = os.path.join(CSRC, "torch_binding.cpp")
    header = os.path.join(REPO_DIR, "include", "nvfp4_b200.h")
    if not force and not _stale(BINDING_PATH, [src, header]) and binding_built_for() == binding_target():
        return BINDING_PATH
    import sysconfig

    import torch
    from torch.utils import cpp_extension
    cuda = os.path.join(os.path.dirname(os.path.dirname(_nvcc())), "include")
    include = cpp_extension.include_paths() + [cuda, sysconfig.get_paths()["include"]]
    tmp = BINDING_PATH + ".tmp"
    # the system compiler, whose C++ runtime is the shared one that libtorch uses: with a
    # second copy linked in, an exception that crosses the two crashes the process
    cxx = next((c for c in ("/usr/bin/g++", shutil.which("g++")) if c and os.path.exists(c)), None)
    if cxx is None:
        raise RuntimeError("g++ not found: the torch binding must be compiled with the system's C++ compiler")
    cmd = [cxx, "-O2", "-std=c++17", "-fPIC", "-shared", src, "-o", tmp,
           f"-DTORCH_EXTENSION_NAME={BINDING_NAME}",
           f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}"]
    for path in include:
        cmd += ["-isystem", path]
    cmd += ["-L" + os.path.join(os.path.dirname(torch.__file__), "lib"), "-lc10", "-lc10_cuda", "-ltorch_cpu",
            "-ltorch", "-ltorch_python", "-L" + LIB_DIR, "-lnvfp4b200", "-Wl,-rpath,$ORIGIN"]
    if verbose:
        print(" ".join(cmd), file=sys.stderr)
    subprocess.run(cmd, check=True)
    os.replace(tmp, BINDING_PATH)
    with open(BINDING_STAMP, "w") as f:
        f.write(binding_target() + "\n")
    return BINDING_PATH


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose=True))
