// The selective state space scan's single step: every env's states go through once.
#pragma once
#include "scan.hpp"

namespace mo {

// A channel's states lie over `lanes` neighbouring lanes (a power of two), V of them each, so that accesses run over the states as they lie; what
// is the channel's own is computed by each of its lanes. A thread goes through STEP_ENVS envs, whose states it has in flight together, with the
// same decays. The states are all there is to move: 8 bytes each, which bound it.
// FAR: the states are more than the last-level cache holds, and go past it.
constexpr int STEP_ENVS = 4;
struct ScanStep {
    MoScan a;
    int lanes;
};

template <class T, int V, bool FAR> __global__ void __launch_bounds__(256) k_scan_step(ScanStep k) {
    const MoScan& a = k.a;
    const int64_t id = block_here() * 256 + threadIdx.x, rest = id / k.lanes, n0 = rest / a.C * STEP_ENVS;
    if (n0 >= a.N) return;
    const int q = (int)(id % k.lanes), c = (int)(rest % a.C), g = c / (a.C / a.G), s0 = q * V;
    const bool live = s0 < a.S;
    typedef Pack<float, V> P;
    P h[STEP_ENVS], A{};
    float* state = a.state_out + (n0 * a.C + c) * a.S + s0;
    const int64_t env = (int64_t)a.C * a.S;
    bool cut[STEP_ENVS];
    T x[STEP_ENVS], dt[STEP_ENVS], z[STEP_ENVS], B[STEP_ENVS][V], C[STEP_ENVS][V];
#pragma unroll
    for (int e = 0; e < STEP_ENVS; e++) {
        const int64_t n = min(n0 + e, a.N - 1);
        cut[e] = a.start && a.start[n];
        if (live && !cut[e]) {
            const P* p = (const P*)(state + (n - n0) * env);
            h[e] = FAR ? streamed(p) : *p;
        }
        const auto at = [&](const MoRows& r) { return ((const T*)r.p)[n * r.sn + c]; };
        x[e] = at(a.x);
        dt[e] = at(a.dt);
        if (a.z.p) z[e] = at(a.z);
        if (live) {
            const T *b = (const T*)a.Bt.p + n * a.Bt.sn + g * a.Bt.sh + s0, *d = (const T*)a.Ct.p + n * a.Ct.sn + g * a.Ct.sh + s0;
#pragma unroll
            for (int v = 0; v < V; v++) {
                B[e][v] = b[v];
                C[e][v] = d[v];
            }
        }
    }
    if (live) A = *(const P*)(a.A + (int64_t)c * a.S + s0);
    const float bias = a.dt_bias ? a.dt_bias[c] : 0.f, D = a.D ? a.D[c] : 0.f;
#pragma unroll
    for (int e = 0; e < STEP_ENVS; e++) {
        if (n0 + e >= a.N) break;
        const float d = softplus(as_f32(dt[e]) + bias).d, u = d * as_f32(x[e]);
        float y = 0.f;
        if (live) {
#pragma unroll
            for (int v = 0; v < V; v++) {
                const float add = u * as_f32(B[e][v]);
                h[e].v[v] = cut[e] ? add : fmaf(exp2_raw(d * (A.v[v] * LOG2E)), h[e].v[v], add);
                y = fmaf(as_f32(C[e][v]), h[e].v[v], y);
            }
            P* p = (P*)(state + e * env);
            if (FAR) stream(p, h[e]);
            else *p = h[e];
        }
        for (int m = 1; m < k.lanes; m *= 2) y += __shfl_xor(y, m);
        if (q) continue;
        if (a.D) y = fmaf(D, as_f32(x[e]), y);
        if (a.z.p) {
            const float zf = as_f32(z[e]);
            y *= zf * sigmoid(zf);
        }
        ((T*)a.out.p)[(n0 + e) * a.out.sn + c] = as<T>(y);
    }
}

template <class T> int scan_step(const MoScan& a, hipStream_t s) {
    const bool wide = a.S % 4 == 0 && (uintptr_t)a.state_out % 16 == 0 && (uintptr_t)a.A % 16 == 0;
    ScanStep k{a, 1};
    while (k.lanes * (wide ? 4 : 1) < a.S) k.lanes *= 2;
    const int64_t envs = (a.N + STEP_ENVS - 1) / STEP_ENVS;
    const dim3 grid = grid_of((envs * a.C * k.lanes + 255) / 256), block(256);
    const bool far = a.N * a.C * a.S * 4 > LAST_LEVEL_CACHE;
    if (wide && far) hipLaunchKernelGGL((k_scan_step<T, 4, true>), grid, block, 0, s, k);
    else if (wide) hipLaunchKernelGGL((k_scan_step<T, 4, false>), grid, block, 0, s, k);
    else hipLaunchKernelGGL((k_scan_step<T, 1, false>), grid, block, 0, s, k);
    return launched("k_scan_step");
}

}  // namespace mo
