"""The operators' hand-written instruction sequences, compiled with operands that are known to be equal: what a sequence has still to read must not be in a
register that it has written."""
import os
import re
import shutil
import subprocess
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
PROBE = """
#include "scan_back.hpp"
using namespace mo;
template <int M> __device__ void sums(float* p) {
    float v[M], x = p[threadIdx.x];
    for (int i = 0; i < M; i++) v[i] = x;
    p[threadIdx.x] = wave_sums<M>(v);
}
__global__ void k_sums4(float* p) { sums<4>(p); }
__global__ void k_sums16(float* p) { sums<16>(p); }
template <int SP> __device__ void set(float* p, const float* b, unsigned cuts) {
    float h[SP], u = p[threadIdx.x], s[SP];
    for (int i = 0; i < SP; i++) { h[i] = u; s[i] = b[i]; }
    if_start_set<1, SP>(cuts, h, u, s);
    for (int i = 0; i < SP; i++) p[threadIdx.x + 64 * i] = h[i];
}
__global__ void k_set4(float* p, const float* b, unsigned cuts) { set<4>(p, b, cuts); }
__global__ void k_set8(float* p, const float* b, unsigned cuts) { set<8>(p, b, cuts); }
"""


def test_sequences_read_their_inputs_before_they_are_written_over(tmp_path):
    if not shutil.which("hipcc"):
        pytest.skip("no hipcc")
    sys.path.insert(0, os.path.join(ROOT, "fast-mario-env_amd"))
    import build_ops
    src, out = tmp_path / "probe.hip", tmp_path / "probe.s"
    src.write_text(PROBE)
    flags = [f for f in build_ops.FLAGS if f not in ("-fPIC", "-Wall")]
    r = subprocess.run(["hipcc", "--offload-arch=gfx950", "--cuda-device-only", "-S", *flags, f"-I{build_ops.CSRC}", str(src), "-o", str(out)], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr[-2000:]
    asm, blocks = out.read_text(), 0
    for name, dpp in (("k_sums4", True), ("k_sums16", True), ("k_set4", False), ("k_set8", False)):
        body = re.search(rf"^_Z\w*{name}\w*:(.*?)s_endpgm", asm, re.S | re.M).group(1)
        for block in re.findall(r";+#ASMSTART(.*?);+#ASMEND", body, re.S):
            written = set()
            for op, args in re.findall(r"(v_\w+) ([^\n;]*)", block):
                to, *of = [a.split()[0] for a in args.split(",")]
                # sums: what comes into the upper lanes (bank mask 0xc) is an input; starts: all are
                if not dpp or "bank_mask:0xc" in args:
                    assert not written & set(of), (name, block)
                written.add(to)
            blocks += len(written) > 1
    assert blocks >= 4                                       # (equal sums may be made once)
