"""Builds libmario_ops.so (the policy's operators: gfx950 code objects + host C ABI) in-tree with hipcc.

    python fast-mario-env_amd/build_ops.py

A library beside libmario_hip.so, whose flags (no fused multiply-adds, scheduling for scalar code) these kernels do not share;
packed FP32 instructions are disabled here too.
"""
from __future__ import annotations

import os
import subprocess
import sys

from build_native import ARCH, HERE, hipcc

SRC = os.path.join(HERE, "csrc", "ops", "mario_ops.hip")
OUT = os.path.join(HERE, "fast_mario_env_amd", "libmario_ops.so")
FLAGS = ["-O3", "-std=c++17", "-fPIC", "-shared", "-fvisibility=hidden", "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
         "-Wall"]


def build(verbose: bool = True) -> str:
    tmp = OUT + ".tmp"
    cmd = [hipcc(), f"--offload-arch={ARCH}", *FLAGS, SRC, "-o", tmp]
    if verbose:
        print("building:", " ".join(cmd), flush=True)
    r = subprocess.run(cmd, capture_output=True, text=True)
    msgs = "\n".join(l for l in (r.stdout + r.stderr).splitlines() if "not a recognized feature" not in l and l.strip())
    if r.returncode != 0:
        raise RuntimeError(f"hipcc failed ({r.returncode}):\n{msgs}")
    if msgs and verbose:
        print(msgs, flush=True)
    os.replace(tmp, OUT)
    return OUT


if __name__ == "__main__":
    print(build())
    sys.exit(0)
