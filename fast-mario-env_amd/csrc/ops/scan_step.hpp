// The selective state space scan's single step: every env's states go through once.
#pragma once
#include "scan.hpp"

namespace mo {

template <class T> __global__ void __launch_bounds__(256) k_scan_step(MoScan a) {
    const int64_t id = block_here() * 256 + threadIdx.x, n = id / a.C;
    if (n >= a.N) return;
    const int c = (int)(id % a.C), g = c / (a.C / a.G);
    const float x = at_row<T>(a.x, 0, n, c), d = softplus(at_row<T>(a.dt, 0, n, c) + (a.dt_bias ? a.dt_bias[c] : 0.f)).d, u = d * x;
    const bool cut = a.start && a.start[n];
    const T *B = (const T*)a.Bt.p + n * a.Bt.sn + g * a.Bt.sh, *C = (const T*)a.Ct.p + n * a.Ct.sn + g * a.Ct.sh;
    float *h = a.state_out + (n * a.C + c) * a.S, y = 0.f;
    for (int s = 0; s < a.S; s++) {
        const float f = u * as_f32(B[s]), v = cut ? f : fmaf(exp2_raw(d * (a.A[(int64_t)c * a.S + s] * LOG2E)), h[s], f);
        h[s] = v;
        y = fmaf(as_f32(C[s]), v, y);
    }
    if (a.D) y = fmaf(a.D[c], x, y);
    if (a.z.p) {
        const float z = at_row<T>(a.z, 0, n, c);
        y *= z * sigmoid(z);
    }
    to_row<T>(a.out, 0, n, c, y);
}

template <class T> int scan_step(const MoScan& a, hipStream_t s) {
    hipLaunchKernelGGL((k_scan_step<T>), grid_of((a.N * a.C + 255) / 256), dim3(256), 0, s, a);
    return launched("k_scan_step");
}

}  // namespace mo
