"""Builds libtorchair_b200.so in-tree with nvcc for sm_100a (the only target)."""
from __future__ import annotations

import os
import shutil
import subprocess
from concurrent.futures import ThreadPoolExecutor

PKG_DIR = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(PKG_DIR, "csrc")
LIB_PATH = os.path.join(PKG_DIR, "libtorchair_b200.so")
TORCH_SOURCE = os.path.join(CSRC, "torch_dense.cpp")
TORCH_LIB_PATH = os.path.join(PKG_DIR, "libtorchair_b200_torch.so")
TORCH_STAMP_PATH = TORCH_LIB_PATH + ".torch"      # the torch it was compiled against: its C++ interface changes with every version
SOURCES = ["api.cu", "quant.cu", "routing.cu", "gmm_i8.cu", "gmm_finalize.cu", "ep_peer.cu", "dense.cu", "checkpoint.cu"]
NVCC_FLAGS = ["-gencode", "arch=compute_100a,code=sm_100a", "-lineinfo", "-O3", "-std=c++17",
              "-Xcompiler", "-fPIC", "-Xcompiler", "-fvisibility=hidden", "--expt-relaxed-constexpr"]


def _nvcc() -> str:
    exe = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    if not os.path.exists(exe):
        raise RuntimeError("nvcc not found; the CUDA toolkit is required to build libtorchair_b200.so")
    return exe


def _stale(target: str, deps) -> bool:
    if not os.path.exists(target):
        return True
    t = os.path.getmtime(target)
    return any(os.path.getmtime(d) > t for d in deps)


def torch_built_against() -> str:
    """The torch that libtorchair_b200_torch.so was compiled against ("" where that is not known)."""
    try:
        with open(TORCH_STAMP_PATH) as f:
            return f.read()
    except FileNotFoundError:
        return ""


def torch_installed() -> str:
    import torch
    return f"{torch.__version__} cxx11abi={int(torch._C._GLIBCXX_USE_CXX11_ABI)}"


def build_torch_library(force: bool = False) -> str:
    """Compiles the PyTorch side of the dense operators against the installed torch and links it to libtorchair_b200.so."""
    api = os.path.join(PKG_DIR, "..", "include", "tab_api.h")
    if not force and torch_built_against() == torch_installed() and not _stale(TORCH_LIB_PATH, [TORCH_SOURCE, api]):
        return TORCH_LIB_PATH
    import torch
    from torch.utils.cpp_extension import include_paths
    lib_dir = os.path.join(os.path.dirname(os.path.abspath(torch.__file__)), "lib")
    cuda_home = os.path.dirname(os.path.dirname(os.path.realpath(_nvcc())))
    cmd = ["g++", "-O2", "-std=c++17", "-fPIC", "-shared", f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}"]
    cmd += [f"-I{d}" for d in include_paths()] + [f"-I{os.path.join(cuda_home, 'include')}", TORCH_SOURCE, "-o", TORCH_LIB_PATH]
    cmd += [f"-L{PKG_DIR}", "-ltorchair_b200", f"-L{lib_dir}", "-ltorch", "-ltorch_cpu", "-ltorch_cuda", "-lc10", "-lc10_cuda",
            "-Wl,-rpath,$ORIGIN"]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"g++ failed on {TORCH_SOURCE}:\n{r.stdout}\n{r.stderr}")
    with open(TORCH_STAMP_PATH, "w") as f:
        f.write(torch_installed())
    return TORCH_LIB_PATH


def build_library(force: bool = False, verbose: bool = False) -> str:
    """Compiles every .cu under csrc/ and links the shared library, then its PyTorch side; returns the former's path."""
    nvcc = _nvcc()
    headers = [os.path.join(CSRC, f) for f in os.listdir(CSRC) if f.endswith((".cuh", ".h"))]
    headers.append(os.path.join(PKG_DIR, "..", "include", "tab_api.h"))
    sources = [s for s in SOURCES if os.path.exists(os.path.join(CSRC, s))]
    objs = []

    def compile_one(src: str) -> str:
        path = os.path.join(CSRC, src)
        obj = os.path.join(CSRC, src[:-3] + ".o")
        if force or _stale(obj, [path] + headers):
            cmd = [nvcc] + NVCC_FLAGS + (["-Xptxas", "-v"] if verbose else []) + ["-c", path, "-o", obj]
            r = subprocess.run(cmd, capture_output=True, text=True)
            if r.returncode != 0:
                raise RuntimeError(f"nvcc failed on {src}:\n{r.stdout}\n{r.stderr}")
            if verbose:
                print(r.stderr)
        return obj

    with ThreadPoolExecutor(max_workers=4) as pool:
        objs = list(pool.map(compile_one, sources))
    if force or _stale(LIB_PATH, objs):
        cmd = [nvcc, "-shared", "-o", LIB_PATH] + objs + ["-cudart", "static"]
        r = subprocess.run(cmd, capture_output=True, text=True)
        if r.returncode != 0:
            raise RuntimeError(f"link failed:\n{r.stdout}\n{r.stderr}")
    build_torch_library(force)
    return LIB_PATH


if __name__ == "__main__":
    import sys
    print(build_library(force="--force" in sys.argv, verbose="-v" in sys.argv))
