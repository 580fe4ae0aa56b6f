"""Build the in-tree CUDA library camoe_b200/libcamoe_wkv7.so for sm_100a, and
camoe_b200/_torch_ops.so, the torch calls of the expert layer and the adapters.

    python -m camoe_b200.build

nvcc cross-compiles without a GPU.  The library links the CUDA runtime
statically, so it loads with or without torch in the process; _torch_ops.so
(csrc/torch_ops.cpp, host code only) is linked against it and against torch.
"""
from __future__ import annotations

import glob
import os
import subprocess
import sys

HERE = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(HERE)
LIB = os.path.join(HERE, "libcamoe_wkv7.so")
TORCH_OPS = os.path.join(HERE, "_torch_ops.so")
TORCH_OPS_SOURCE = os.path.join(HERE, "csrc", "torch_ops.cpp")
GENCODE = "arch=compute_100a,code=sm_100a"


def sources() -> list[str]:
    return sorted(glob.glob(os.path.join(HERE, "csrc", "*.cu")))


def nvcc_command(out: str = LIB, extra: list[str] | None = None) -> list[str]:
    nvcc = os.environ.get("NVCC", "nvcc")
    return [nvcc, "-gencode", GENCODE, "-O3", "-lineinfo", "-std=c++17",
            "-Xcompiler", "-fPIC", "-shared", "-I", os.path.join(ROOT, "include"),
            *(extra or []), "-o", out, *sources()]


def torch_ops_command(out: str = TORCH_OPS) -> list[str]:
    import sysconfig

    import torch
    root = os.path.dirname(os.path.abspath(torch.__file__))
    cuda = os.environ.get("CUDA_HOME", "/usr/local/cuda")
    include = [os.path.join(root, "include"), os.path.join(root, "include", "torch", "csrc", "api", "include"),
               os.path.join(cuda, "include"), sysconfig.get_paths()["include"], os.path.join(ROOT, "include")]
    return [os.environ.get("CXX", "g++"), "-O2", "-std=c++17", "-fPIC", "-shared",
            "-DTORCH_EXTENSION_NAME=_torch_ops",
            f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
            *(x for i in include for x in ("-isystem", i)), TORCH_OPS_SOURCE, "-o", out,
            "-L", HERE, "-l:libcamoe_wkv7.so", "-Wl,-rpath,$ORIGIN", "-L", os.path.join(root, "lib"),
            "-ltorch_python", "-ltorch", "-ltorch_cpu", "-ltorch_cuda", "-lc10", "-lc10_cuda"]


def up_to_date(out: str = LIB) -> bool:
    if not os.path.exists(out):
        return False
    t = os.path.getmtime(out)
    if out == TORCH_OPS:
        return all(os.path.getmtime(d) <= t for d in
                   [TORCH_OPS_SOURCE, os.path.join(ROOT, "include", "camoe_experts.h")])
    deps = sources() + glob.glob(os.path.join(HERE, "csrc", "*.cuh")) + \
        glob.glob(os.path.join(ROOT, "include", "*.h"))
    return all(os.path.getmtime(d) <= t for d in deps)


def build(force: bool = False, verbose: bool = False) -> str:
    if force or not up_to_date():
        cmd = nvcc_command(extra=["-Xptxas", "-v"] if verbose else None)
        subprocess.run(cmd, check=True)
    if force or not up_to_date(TORCH_OPS):
        subprocess.run(torch_ops_command(), check=True)
    return LIB


if __name__ == "__main__":
    build(force="--force" in sys.argv, verbose="-v" in sys.argv)
    print(LIB)
