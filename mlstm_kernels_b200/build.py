"""Build recipe for libmlstm_b200.so (plain nvcc, sm_100a only) and for _host.so, the native host side of the PyTorch
functions (plain g++ against the installed PyTorch); both in-tree next to this file.

    python -m mlstm_kernels_b200.build          # incremental
    python -m mlstm_kernels_b200.build --force  # rebuild everything

nvcc cross-compiles without a GPU.  Objects go to mlstm_kernels_b200/build/ (git-ignored).
"""

from __future__ import annotations

import os
import shutil
import subprocess
import sys
import sysconfig
from concurrent.futures import ThreadPoolExecutor

PKG = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(PKG, "csrc")
OBJ = os.path.join(PKG, "build")
LIB = os.path.join(PKG, "libmlstm_b200.so")
HOST = os.path.join(PKG, "_host.so")
SOURCES = ["api.cu", "gates.cu", "step.cu", "chunkwise_simt.cu", "chunkwise_sm100.cu", "chunkwise_bw_sm100.cu", "noalloc.cu",
           "api_layers.cu", "layer_norm.cu", "short_conv.cu", "ssm_fw.cu", "ssm_bw.cu"]
HOST_SOURCES = ["host.cpp", "host_layers.cpp"]
NVCC_FLAGS = [
    "-gencode", "arch=compute_100a,code=sm_100a", "-lineinfo", "-O3", "-std=c++17",
    "--use_fast_math=false", "-Xcompiler", "-fPIC", "-Xcompiler", "-fvisibility=hidden",
    "--expt-relaxed-constexpr",
]


def _nvcc() -> str:
    cand = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    if not os.path.exists(cand):
        raise RuntimeError("nvcc not found: the CUDA toolkit is required to build libmlstm_b200.so")
    return cand


def _deps_mtime() -> float:
    hdrs = [os.path.join(CSRC, f) for f in os.listdir(CSRC) if f.endswith((".cuh", ".h"))]
    hdrs.append(os.path.join(os.path.dirname(PKG), "include", "mlstm_b200.h"))
    return max(os.path.getmtime(h) for h in hdrs)


def _host_commands() -> tuple[list[list[str]], list[str]]:
    """What compiles each source of _host.so, and what links them."""
    import torch
    from torch.utils import cpp_extension

    cuda = os.path.dirname(os.path.dirname(_nvcc()))
    inc = [*cpp_extension.include_paths(), os.path.join(cuda, "include"), sysconfig.get_paths()["include"]]
    lib = os.path.join(os.path.dirname(torch.__file__), "lib")
    objs = [os.path.join(OBJ, s.replace(".cpp", ".o")) for s in HOST_SOURCES]
    compiles = [["g++", "-O2", "-std=c++17", "-fPIC", "-fvisibility=hidden",
                 f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}", *(f"-I{p}" for p in inc),
                 "-c", os.path.join(CSRC, s), "-o", o] for s, o in zip(HOST_SOURCES, objs)]
    link = ["g++", "-shared", *objs, "-o", HOST, f"-L{PKG}", "-l:libmlstm_b200.so", "-Wl,-rpath,$ORIGIN",
            f"-L{lib}", "-ltorch_python", "-ltorch", "-ltorch_cuda", "-ltorch_cpu", "-lc10_cuda", "-lc10"]
    return compiles, link


def build(force: bool = False, verbose: bool = False) -> str:
    os.makedirs(OBJ, exist_ok=True)
    nvcc = _nvcc()
    hdr_t = _deps_mtime()
    jobs = []
    objs = []
    for src in SOURCES:
        s = os.path.join(CSRC, src)
        o = os.path.join(OBJ, src.replace(".cu", ".o"))
        objs.append(o)
        if force or not os.path.exists(o) or os.path.getmtime(o) < max(os.path.getmtime(s), hdr_t):
            flags = [f for f in NVCC_FLAGS if f != "--use_fast_math=false"]
            cmd = [nvcc, *flags, "-c", s, "-o", o]
            if verbose:
                cmd.insert(1, "-Xptxas=-v")
            jobs.append(cmd)

    def run(cmd):
        r = subprocess.run(cmd, capture_output=True, text=True)
        if r.returncode != 0:
            raise RuntimeError("build failed:\n" + " ".join(cmd) + "\n" + r.stdout + r.stderr)
        return r.stderr

    if jobs:
        with ThreadPoolExecutor(max_workers=min(len(jobs), os.cpu_count() or 1)) as ex:
            for out in ex.map(run, jobs):
                if verbose and out:
                    print(out)
    if jobs or not os.path.exists(LIB):
        run([nvcc, "-shared", "-o", LIB, *objs, "-gencode", "arch=compute_100a,code=sm_100a", "-lcuda"])
    host_t = max(hdr_t, *(os.path.getmtime(os.path.join(CSRC, s)) for s in HOST_SOURCES))
    if force or not os.path.exists(HOST) or os.path.getmtime(HOST) < host_t:
        compiles, link = _host_commands()
        with ThreadPoolExecutor(max_workers=len(compiles)) as ex:
            list(ex.map(run, compiles))
        run(link)
    return LIB


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose="-v" in sys.argv))
