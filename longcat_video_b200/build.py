"""Build ``liblcbsa.so`` (the CUDA kernels plus the C ABI of ``include/lcbsa.h``) in-tree with nvcc, and ``_binding-<torch and Python>.so``,
the Python functions and autograd nodes of ``csrc/binding.cpp``, with g++ against this Python's torch.

    python -m longcat_video_b200.build [--force]

The library is compiled for sm_100a only and lands next to the sources
(``longcat_video_b200/csrc/liblcbsa.so``).
"""
from __future__ import annotations

import concurrent.futures
import os
import shutil
import subprocess
import sys

CSRC = os.path.join(os.path.dirname(os.path.abspath(__file__)), "csrc")
LIB = os.path.join(CSRC, "liblcbsa.so")
SOURCES = ["api.cu", "pool.cu", "select.cu", "select_gemm.cu", "select_cdf.cu", "attn_mma.cu", "attn_tc.cu", "attn_tc128.cu", "attn_bwd.cu", "attn_bwd_tc.cu", "noalloc.cu", "norm_rope.cu",
           "rotary.cu", "dense_plan.cu", "dense_few.cu", "dense_tc.cu", "dense_bwd_tc.cu"]
HEADERS = ["common.cuh", "select_common.cuh", "tc_common.cuh", "mma_common.cuh", "dense_common.cuh", os.path.join("..", "..", "include", "lcbsa.h")]
NVCC_FLAGS = ["-gencode", "arch=compute_100a,code=sm_100a", "-lineinfo", "-O3", "-std=c++17",
              "-Xcompiler", "-fPIC", "--expt-relaxed-constexpr"]


def _nvcc() -> str:
    exe = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    if not os.path.exists(exe):
        raise RuntimeError("nvcc not found; liblcbsa.so cannot be built")
    return exe


def _sources():
    return [s for s in SOURCES if os.path.exists(os.path.join(CSRC, s))]


def _stale() -> bool:
    if not os.path.exists(LIB):
        return True
    t = os.path.getmtime(LIB)
    deps = [os.path.join(CSRC, s) for s in _sources()] + [os.path.join(CSRC, h) for h in HEADERS]
    return any(os.path.getmtime(d) > t for d in deps)


def _build_binding(force: bool) -> None:
    src, header = os.path.join(CSRC, "binding.cpp"), os.path.join(CSRC, "..", "..", "include", "lcbsa.h")
    import sysconfig

    import torch

    from ._lib import binding_path
    binding = binding_path()  # another one for another torch or Python
    if not force and os.path.exists(binding) and os.path.getmtime(binding) > max(os.path.getmtime(p) for p in (src, header)):
        return
    root = os.path.dirname(torch.__file__)
    include = [os.path.join(root, "include"), os.path.join(root, "include", "torch", "csrc", "api", "include"), sysconfig.get_paths()["include"],
               os.path.join(os.path.dirname(os.path.dirname(_nvcc())), "include")]
    lib = os.path.join(root, "lib")
    cmd = ["g++", "-std=c++17", "-O2", "-fPIC", "-shared", f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
           *(f"-isystem{p}" for p in include), src, "-o", binding, f"-L{CSRC}", "-l:liblcbsa.so", "-Wl,-rpath,$ORIGIN", f"-L{lib}", "-ltorch",
           "-ltorch_cpu", "-ltorch_cuda", "-ltorch_python", "-lc10", "-lc10_cuda"]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"g++ failed on binding.cpp:\n{r.stdout}\n{r.stderr}")


def build(force: bool = False, verbose: bool = False) -> str:
    if not force and not _stale():
        _build_binding(force)
        return LIB
    nvcc = _nvcc()
    objs = []

    def compile_one(src):
        obj = os.path.join(CSRC, src[:-3] + ".o")
        cmd = [nvcc, *NVCC_FLAGS, "-c", os.path.join(CSRC, src), "-o", obj]
        if verbose:
            cmd.insert(1, "-Xptxas=-v")
        r = subprocess.run(cmd, capture_output=True, text=True)
        if r.returncode != 0:
            raise RuntimeError(f"nvcc failed on {src}:\n{r.stdout}\n{r.stderr}")
        if verbose:
            sys.stderr.write(r.stderr)
        return obj

    with concurrent.futures.ThreadPoolExecutor(max_workers=8) as ex:
        objs = list(ex.map(compile_one, _sources()))
    cmd = [nvcc, "-shared", "-o", LIB, *objs, "-lcudart"]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"link failed:\n{r.stdout}\n{r.stderr}")
    _build_binding(force)
    return LIB


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose="-v" in sys.argv))
