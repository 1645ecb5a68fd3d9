"""Builds the policy's operators in-tree:

- libmario_ops.so with hipcc: gfx950 code objects + host C ABI (include/mario_ops.h). A library beside libmario_hip.so, whose flags
  (no fused multiply-adds, scheduling for scalar code) these kernels do not share; packed FP32 instructions are disabled here too.
- _mario_ops_torch, the extension module that calls it on torch tensors, with g++ against the installed torch.

    python fast-mario-env_amd/build_ops.py
"""
from __future__ import annotations

import os
import shutil
import subprocess
import sys
import sysconfig

from build_native import ARCH, HERE, hipcc

CSRC = os.path.join(HERE, "csrc", "ops")
PACKAGE = os.path.join(HERE, "fast_mario_env_amd")
OUT = os.path.join(PACKAGE, "libmario_ops.so")
EXTENSION = os.path.join(PACKAGE, "_mario_ops_torch" + sysconfig.get_config_var("EXT_SUFFIX"))
FLAGS = ["-O3", "-std=c++17", "-fPIC", "-shared", "-fvisibility=hidden", "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
         "-Wall"]


def _run(cmd, out, verbose):
    cmd = [*cmd, "-o", out + ".tmp"]
    if verbose:
        print("building:", " ".join(cmd), flush=True)
    r = subprocess.run(cmd, capture_output=True, text=True)
    msgs = "\n".join(l for l in (r.stdout + r.stderr).splitlines() if "not a recognized feature" not in l and l.strip())
    if r.returncode != 0:
        raise RuntimeError(f"{cmd[0]} failed ({r.returncode}):\n{msgs}")
    if msgs and verbose:
        print(msgs, flush=True)
    os.replace(out + ".tmp", out)


def build(verbose: bool = True) -> str:
    _run([hipcc(), f"--offload-arch={ARCH}", *FLAGS, os.path.join(CSRC, "mario_ops.hip")], OUT, verbose)
    import torch
    from torch.utils.cpp_extension import include_paths
    lib, rocm = os.path.join(os.path.dirname(torch.__file__), "lib"), os.path.dirname(os.path.dirname(os.path.realpath(hipcc())))
    headers = [*include_paths(), os.path.join(rocm, "include"), "/opt/rocm/include", sysconfig.get_paths()["include"]]
    _run([os.environ.get("CXX") or shutil.which("g++") or "c++", "-O2", "-std=c++17", "-fPIC", "-shared", "-fvisibility=hidden",
          "-D__HIP_PLATFORM_AMD__=1", "-DUSE_ROCM=1", f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
          *(flag for h in headers for flag in ("-isystem", h)), os.path.join(CSRC, "torch_ops.cpp"), f"-L{lib}", f"-L{PACKAGE}",
          "-lmario_ops", "-lc10", "-lc10_hip", "-ltorch", "-ltorch_cpu", "-ltorch_python", "-Wl,-rpath,$ORIGIN"], EXTENSION, verbose)
    return OUT


if __name__ == "__main__":
    print(build())
    sys.exit(0)
