"""Build libytm.so in-tree for sm_100a (B200).

    python -m ytm_b200.build          # or ytm_b200.build.build()

nvcc cross-compiles without a GPU.  The library lands next to this file so it
travels with the source tree; nothing is installed into site-packages.
"""
from __future__ import annotations

import glob
import os
import subprocess
import sys

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
LIB = os.path.join(HERE, "libytm.so")
NVCC_FLAGS = [
    "-O3", "-std=c++17", "-lineinfo",
    "-gencode", "arch=compute_100a,code=sm_100a",
    "-Xcompiler", "-fPIC", "-shared",
    "--expt-relaxed-constexpr", "--threads", "0",
]


def nccl_flags() -> list[str]:
    """Include/link flags for NCCL: the headers of the NCCL wheel that torch
    loads (same version at run time), else the system's."""
    try:
        import nvidia.nccl as n  # the wheel torch depends on
        base = os.path.dirname(n.__file__) if getattr(n, "__file__", None) else list(n.__path__)[0]
        inc, lib = os.path.join(base, "include"), os.path.join(base, "lib")
        if os.path.exists(os.path.join(inc, "nccl.h")):
            return ["-I" + inc, "-L" + lib, "-l:libnccl.so.2"]
    except ImportError:
        pass
    return ["-lnccl"]


def sources() -> list[str]:
    return sorted(glob.glob(os.path.join(CSRC, "*.cu")))


BIND = os.path.join(HERE, "_answers.so")


def _bind_stale() -> bool:
    deps = [os.path.join(CSRC, "answers_bind.cpp"), os.path.join(HERE, "..", "include", "ytm.h"), LIB]
    return not os.path.exists(BIND) or any(os.path.getmtime(d) > os.path.getmtime(BIND) for d in deps)


def build_bind(force: bool = False, verbose: bool = False) -> str:
    """The Python entry points of ytm_b200.answers over libytm.so."""
    if not force and not _bind_stale():
        return BIND
    import sysconfig

    import torch
    from torch.utils.cpp_extension import include_paths
    torch_lib = os.path.join(os.path.dirname(torch.__file__), "lib")
    cuda = os.path.join(os.environ.get("CUDA_HOME", "/usr/local/cuda"), "include")
    cmd = [os.environ.get("CXX", "g++"), "-O2", "-std=c++17", "-shared", "-fPIC",
           f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}", os.path.join(CSRC, "answers_bind.cpp"),
           *("-I" + i for i in (*include_paths(), sysconfig.get_paths()["include"], cuda)), "-L" + torch_lib,
           "-ltorch_python", "-ltorch", "-ltorch_cpu", "-lc10", "-lc10_cuda", "-L" + HERE, "-l:libytm.so",
           "-Wl,-rpath,$ORIGIN", "-Wl,-rpath," + torch_lib, "-o", BIND + ".tmp"]
    if verbose:
        print(" ".join(cmd), file=sys.stderr)
    subprocess.run(cmd, check=True)
    os.replace(BIND + ".tmp", BIND)
    return BIND


def _stale() -> bool:
    if not os.path.exists(LIB):
        return True
    t = os.path.getmtime(LIB)
    deps = sources() + glob.glob(os.path.join(CSRC, "*.cuh")) + [
        os.path.join(HERE, "..", "include", "ytm.h"), __file__]
    return any(os.path.getmtime(d) > t for d in deps if os.path.exists(d))


def build(force: bool = False, verbose: bool = False, extra: list[str] | None = None) -> str:
    if not force and not _stale():
        build_bind(verbose=verbose)
        return LIB
    nvcc = os.environ.get("NVCC", "nvcc")
    tmp = LIB + ".tmp"
    cmd = [nvcc, *NVCC_FLAGS, *(extra or []), *sources(), *nccl_flags(), "-o", tmp]
    if verbose:
        print(" ".join(cmd), file=sys.stderr)
    subprocess.run(cmd, check=True)
    os.replace(tmp, LIB)
    build_bind(verbose=verbose)
    return LIB


PROBE_SRC = os.path.join(HERE, "..", "bench_probe.cu")
PROBE_LIB = os.path.join(HERE, "..", "bench_probe.so")


def build_probe(force: bool = False) -> str | None:
    """bench.py's LOP3 throughput probe (not part of libytm), beside bench.py."""
    if not os.path.exists(PROBE_SRC):
        return None
    if not force and os.path.exists(PROBE_LIB) and os.path.getmtime(PROBE_LIB) >= os.path.getmtime(PROBE_SRC):
        return PROBE_LIB
    nvcc = os.environ.get("NVCC", "nvcc")
    subprocess.run([nvcc, *NVCC_FLAGS, PROBE_SRC, "-o", PROBE_LIB + ".tmp"], check=True)
    os.replace(PROBE_LIB + ".tmp", PROBE_LIB)
    return PROBE_LIB


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose=True,
                extra=["-Xptxas", "-v"] if "--ptxas" in sys.argv else None))
