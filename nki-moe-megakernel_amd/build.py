"""Build libmkd.so (the gfx950 HIP library behind the C ABI in include/mkd.h) and
_mkd_torch.so (the native torch boundary of some operators, on top of it).

One hipcc invocation per source into objects under _build/, then one link; the
torch boundary is host code, compiled by g++ against torch's headers.
Sources are compiled for gfx950 only, with packed-fp32 code generation
disabled.  Run as ``python nki-moe-megakernel_amd/build.py`` or through
``__graft_entry__.build()``.
"""
from __future__ import annotations

import concurrent.futures as cf
import os
import subprocess
import sys

PKG_DIR = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(PKG_DIR, "csrc")
BUILD_DIR = os.path.join(PKG_DIR, "_build")
LIB_PATH = os.path.join(PKG_DIR, "libmkd.so")
TORCH_LIB_PATH = os.path.join(PKG_DIR, "_mkd_torch.so")
SOURCES = ["capi.hip", "gemm.hip", "norm.hip", "attn_mfma.hip", "moe.hip",
           "misc.hip", "mx.hip", "gemm_tile.hip", "layer_mk.hip", "qkv_norm.hip", "gemm_mid.hip",
           "attn_kvfmt.hip", "attn_stream.hip", "gemm_w8.hip", "attn_prefill.hip",
           "kv_append.hip", "attn_shared.hip", "sample.hip"]
HIPCC = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")
ARCH = "gfx950"

COMMON_FLAGS = [
    f"--offload-arch={ARCH}", "-O3", "-std=c++17", "-fPIC",
    "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
    "-Wno-unused-result", "-Werror=uninitialized", "-I", os.path.join(PKG_DIR, "..", "include"),
]


def _compile(src: str) -> str:
    obj = os.path.join(BUILD_DIR, os.path.splitext(src)[0] + ".o")
    cmd = [HIPCC, *COMMON_FLAGS, "-c", os.path.join(CSRC, src), "-o", obj]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"hipcc failed for {src}:\n{r.stderr[-6000:]}")
    return obj


def _compile_torch() -> str:
    import sysconfig
    import torch
    inc = os.path.join(os.path.dirname(torch.__file__), "include")
    obj = os.path.join(BUILD_DIR, "torch_ops.o")
    cmd = ["g++", "-O2", "-std=c++17", "-fPIC", "-D__HIP_PLATFORM_AMD__=1", "-DUSE_ROCM=1",
           f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}", "-isystem", inc, "-isystem",
           os.path.join(inc, "torch", "csrc", "api", "include"), "-isystem", "/opt/rocm/include", "-isystem",
           sysconfig.get_paths()["include"], "-I", os.path.join(PKG_DIR, "..", "include"),
           "-c", os.path.join(CSRC, "torch_ops.cpp"), "-o", obj]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"g++ failed for torch_ops.cpp:\n{r.stderr[-6000:]}")
    return obj


def _link_torch(obj: str) -> None:
    import torch
    libs = os.path.join(os.path.dirname(torch.__file__), "lib")
    tmp = TORCH_LIB_PATH + ".tmp"
    cmd = ["g++", "-shared", "-fPIC", obj, "-o", tmp, "-L", PKG_DIR, "-l:libmkd.so", "-Wl,-rpath,$ORIGIN", "-L", libs,
           "-lc10", "-ltorch_cpu", "-ltorch_python", "-lc10_hip", "-ltorch_hip"]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"link of _mkd_torch.so failed:\n{r.stderr[-6000:]}")
    os.replace(tmp, TORCH_LIB_PATH)


def build(verbose: bool = True) -> str:
    os.makedirs(BUILD_DIR, exist_ok=True)
    srcs = [s for s in SOURCES if os.path.exists(os.path.join(CSRC, s))]
    with cf.ThreadPoolExecutor(max_workers=min(len(srcs), 4)) as ex:
        torch_obj = ex.submit(_compile_torch)
        objs = list(ex.map(_compile, srcs))
    tmp = LIB_PATH + ".tmp"
    cmd = [HIPCC, f"--offload-arch={ARCH}", "-shared", "-fPIC", "-Wl,-soname,libmkd.so", *objs, "-o", tmp]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"link failed:\n{r.stderr[-6000:]}")
    os.replace(tmp, LIB_PATH)
    _link_torch(torch_obj.result())
    if verbose:
        print(f"built {LIB_PATH} and {TORCH_LIB_PATH}")
    return LIB_PATH


if __name__ == "__main__":
    build()
    sys.exit(0)
