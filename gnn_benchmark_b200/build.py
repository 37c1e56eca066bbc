"""Build libgnnagg.so (the C-ABI CUDA library, sm_100a, nvcc) and _torch_ops.so (the torch front end of the
low-precision operators over that C ABI, g++) in-tree.

usage: python -m gnn_benchmark_b200.build [--force] [--verbose]
"""
import glob
import os
import subprocess
import sys

PKG_DIR = os.path.dirname(os.path.abspath(__file__))
REPO_ROOT = os.path.dirname(PKG_DIR)
CSRC = os.path.join(PKG_DIR, "csrc")
LIB_PATH = os.path.join(PKG_DIR, "libgnnagg.so")
OPS_SOURCE = os.path.join(CSRC, "torch", "ops.cpp")
OPS_PATH = os.path.join(PKG_DIR, "_torch_ops.so")

NVCC_FLAGS = [
    "-O3",
    "-std=c++17",
    "-gencode", "arch=compute_100a,code=sm_100a",
    "-lineinfo",
    "-Xcompiler", "-fPIC",
    "--shared",
    "--threads", "0",  # as many files at once as the machine has cores
    "-ccbin", "/usr/bin/g++",
]


def sources():
    return sorted(glob.glob(os.path.join(CSRC, "*.cu")))


def _stale() -> bool:
    if not os.path.isfile(LIB_PATH):
        return True
    t = os.path.getmtime(LIB_PATH)
    deps = sources() + glob.glob(os.path.join(CSRC, "*.cuh")) + glob.glob(os.path.join(REPO_ROOT, "include", "*.h"))
    return any(os.path.getmtime(d) > t for d in deps)


def _build_ops(force: bool) -> None:
    """Compile the torch front end; it links libgnnagg.so from its own folder."""
    deps = (OPS_SOURCE, os.path.join(REPO_ROOT, "include", "gnnagg.h"))
    if not force and os.path.isfile(OPS_PATH) and all(os.path.getmtime(d) <= os.path.getmtime(OPS_PATH) for d in deps):
        return
    import sysconfig

    import torch
    from torch.utils import cpp_extension

    cuda = os.path.dirname(os.path.dirname(os.environ.get("NVCC", "/usr/local/cuda/bin/nvcc")))
    include = cpp_extension.include_paths() + [os.path.join(cuda, "include"), sysconfig.get_paths()["include"],
                                               os.path.join(REPO_ROOT, "include")]
    libs = os.path.join(os.path.dirname(torch.__file__), "lib")
    cmd = ["/usr/bin/g++", "-O2", "-std=c++17", "-fPIC", "-shared", "-DTORCH_EXTENSION_NAME=_torch_ops",
           "-DTORCH_API_INCLUDE_EXTENSION_H", f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}"]
    for d in include:
        cmd += ["-isystem", d]
    cmd += [OPS_SOURCE, "-o", OPS_PATH, "-L", PKG_DIR, "-l:libgnnagg.so", "-L", libs, "-ltorch", "-ltorch_cpu", "-ltorch_cuda",
            "-lc10", "-lc10_cuda", "-ltorch_python", "-Wl,-rpath,$ORIGIN", f"-Wl,-rpath,{libs}"]
    subprocess.run(cmd, check=True)


def build(force: bool = False, verbose: bool = False) -> str:
    """Compile every .cu under csrc/ into libgnnagg.so and csrc/torch into _torch_ops.so; returns the former's path."""
    if force or _stale():
        _build_lib(verbose)
    _build_ops(force)
    return LIB_PATH


def _build_lib(verbose: bool) -> None:
    nvcc = os.environ.get("NVCC", "/usr/local/cuda/bin/nvcc")
    cmd = [nvcc] + NVCC_FLAGS + ["-I", os.path.join(REPO_ROOT, "include"), "-I", CSRC]
    if verbose:
        cmd += ["-Xptxas", "-v"]
    cmd += sources() + ["-o", LIB_PATH]
    subprocess.run(cmd, check=True)


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose="--verbose" in sys.argv))
