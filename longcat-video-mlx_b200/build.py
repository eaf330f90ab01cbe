"""Build the BSA engine's C-ABI shared library in-tree for sm_100a.

    python longcat-video-mlx_b200/build.py [--verbose]

Output: longcat-video-mlx_b200/longcat_video/_lib/libbsa_b200.so and _dense_ops.so, the torch binding of its
dense side (git-ignored; they travel with the source tree).  nvcc cross-compiles, so this runs on a machine without a GPU.
"""

from __future__ import annotations

import os
import shutil
import subprocess
import sys
import sysconfig

HERE = os.path.dirname(os.path.abspath(__file__))
REPO = os.path.dirname(HERE)
CSRC = os.path.join(HERE, "csrc")
LIB_DIR = os.path.join(HERE, "longcat_video", "_lib")
LIB_PATH = os.path.join(LIB_DIR, "libbsa_b200.so")
SOURCES = ["bsa_capi.cu", "bsa_attn.cu", "bsa_score.cu", "bsa_route.cu", "bsa_noalloc.cu", "bsa_xfer.cu",
           "bsa_dense_capi.cu", "bsa_normrope.cu", "bsa_ranges.cu", "bsa_kv8.cu", "bsa_dense.cu", "bsa_dense_bwd.cu"]
HEADERS = ["bsa_ptx.cuh", "bsa_kernels.h", "bsa_select.cuh", "bsa_dense.h", "bsa_dense.cuh", "bsa_rows.cuh"]


OPS_PATH = os.path.join(LIB_DIR, "_dense_ops.so")  # Python binding of the dense side
OPS_SOURCE = os.path.join(CSRC, "dense_ops.cpp")


def nvcc_path() -> str:
    for cand in (os.environ.get("NVCC"), shutil.which("nvcc"), "/usr/local/cuda/bin/nvcc"):
        if cand and os.path.exists(cand):
            return cand
    raise RuntimeError("nvcc not found")


def _stale() -> bool:
    if not os.path.exists(LIB_PATH):
        return True
    t = os.path.getmtime(LIB_PATH)
    deps = [os.path.join(CSRC, f) for f in SOURCES + HEADERS] + [os.path.join(REPO, "include", "bsa_b200.h"),
                                                                  os.path.abspath(__file__)]
    return any(os.path.getmtime(d) > t for d in deps if os.path.exists(d))


def build_ops(force: bool = False) -> str:
    """The torch binding of the dense side: host code only, compiled against this interpreter's torch."""
    deps = (OPS_SOURCE, os.path.join(REPO, "include", "bsa_b200.h"), os.path.abspath(__file__))
    if not force and os.path.exists(OPS_PATH) and all(os.path.getmtime(d) <= os.path.getmtime(OPS_PATH) for d in deps):
        return OPS_PATH
    os.makedirs(LIB_DIR, exist_ok=True)
    import torch

    root = os.path.join(os.path.dirname(torch.__file__), "include")
    cuda = os.path.join(os.path.dirname(os.path.dirname(nvcc_path())), "include")
    include = [root, os.path.join(root, "torch", "csrc", "api", "include"), sysconfig.get_paths()["include"], cuda]
    cmd = ["g++", "-O2", "-std=c++17", "-fPIC", "-shared", "-DTORCH_EXTENSION_NAME=_dense_ops",
           f"-D_GLIBCXX_USE_CXX11_ABI={int(torch.compiled_with_cxx11_abi())}"]
    cmd += [x for i in include for x in ("-isystem", i)] + ["-o", OPS_PATH + ".tmp", OPS_SOURCE]
    cmd += ["-L" + os.path.join(os.path.dirname(torch.__file__), "lib"), "-lc10", "-lc10_cuda", "-ltorch_cpu", "-ltorch",
            "-ltorch_python", "-ldl"]
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError(f"g++ failed:\n{res.stdout}\n{res.stderr}")
    os.replace(OPS_PATH + ".tmp", OPS_PATH)
    return OPS_PATH


def build(force: bool = False, verbose: bool = False) -> str:
    build_ops(force)
    if not force and not _stale():
        return LIB_PATH
    os.makedirs(LIB_DIR, exist_ok=True)
    cmd = [nvcc_path(), "-gencode", "arch=compute_100a,code=sm_100a", "-O3", "-lineinfo", "-std=c++17", "--threads", "0",
           "-shared", "-Xcompiler", "-fPIC", "-I", os.path.join(REPO, "include"),
           "-o", LIB_PATH + ".tmp"] + [os.path.join(CSRC, f) for f in SOURCES]
    if verbose:
        cmd += ["-Xptxas", "-v"]
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError(f"nvcc failed:\n{res.stdout}\n{res.stderr}")
    if verbose:
        sys.stderr.write(res.stderr)
    os.replace(LIB_PATH + ".tmp", LIB_PATH)
    return LIB_PATH


if __name__ == "__main__":
    print(build(force="--stale" not in sys.argv, verbose="--verbose" in sys.argv))
