"""Compiles the HIP libraries khq/libkhq_hip.so and khq/libkhq_paged.so (the
paged cache, linked to the first) for gfx950 with hipcc, and the Python module
khq/_paged.so (the paged calls' argument checks) with the host compiler."""
from __future__ import annotations

import os
import subprocess
import sys
import sysconfig

PKG_DIR = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(PKG_DIR)
REPO = os.path.dirname(ROOT)
CSRC = os.path.join(ROOT, "csrc")
INCLUDE = os.path.join(REPO, "include")
LIB_NAME = "libkhq_hip.so"
LIB_PATH = os.path.join(PKG_DIR, LIB_NAME)
SOURCES = ["khq_kernels.hip", "khq_attn_ws.hip", "khq_finish.hip", "khq_prefill.hip", "khq_dump.hip", "khq_calib.hip",
           "khq_capi.cpp", "khq_layer.cpp"]
PAGED_LIB_NAME = "libkhq_paged.so"
PAGED_LIB_PATH = os.path.join(PKG_DIR, PAGED_LIB_NAME)
PAGED_SOURCES = ["khq_paged.hip", "khq_paged_attn.hip", "khq_paged_capi.cpp"]
PAGED_CALLS_PATH = os.path.join(PKG_DIR, "_paged.so")

CXX = os.environ.get("CXX", "g++")
HIPCC = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")
ARCH = os.environ.get("KHQ_OFFLOAD_ARCH", "gfx950")

# -ffp-contract=off: only explicit fmaf() fuses (bit-exact compress codes).
# -packed-fp32-ops disabled: no v_pk_{add,mul,fma}_f32 in device code.
FLAGS = [
    f"--offload-arch={ARCH}", "-O3", "-std=c++17", "-fPIC", "-shared",
    "-ffp-contract=off", "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
    "-Wno-unused-command-line-argument",
]


def _run(cmd, path: str, verbose: bool) -> None:
    cmd = [*cmd, "-o", path + ".tmp"]
    if verbose:
        print(" ".join(cmd), flush=True)
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        sys.stderr.write(res.stdout + res.stderr)
        raise RuntimeError(f"{cmd[0]} failed ({res.returncode}) building {os.path.basename(path)}")
    os.replace(path + ".tmp", path)


def _compile(sources, path: str, extra, verbose: bool) -> None:
    _run([HIPCC, *FLAGS, "-I", INCLUDE, "-I", CSRC, *[os.path.join(CSRC, s) for s in sources],
          *extra], path, verbose)


def _compile_calls(verbose: bool) -> None:
    import torch

    base = os.path.dirname(torch.__file__)
    rocm = os.path.dirname(os.path.dirname(os.path.realpath(HIPCC)))
    _run([CXX, "-O2", "-std=c++17", "-fPIC", "-shared", "-D__HIP_PLATFORM_AMD__=1",
          f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}", "-I", INCLUDE,
          "-isystem", os.path.join(rocm, "include"), "-isystem", os.path.join(base, "include"),
          "-isystem", sysconfig.get_paths()["include"], os.path.join(CSRC, "khq_paged_py.cpp"),
          "-L", PKG_DIR, f"-l:{PAGED_LIB_NAME}", "-Wl,-rpath,$ORIGIN",
          "-L", os.path.join(base, "lib"), "-ltorch_python", "-lc10"], PAGED_CALLS_PATH, verbose)


def build(verbose: bool = False) -> str:
    _compile(SOURCES, LIB_PATH, [], verbose)
    _compile(PAGED_SOURCES, PAGED_LIB_PATH,
             ["-L", PKG_DIR, f"-l:{LIB_NAME}", "-Wl,-rpath,$ORIGIN"], verbose)
    _compile_calls(verbose)
    return LIB_PATH


if __name__ == "__main__":
    print(build(verbose=True))
