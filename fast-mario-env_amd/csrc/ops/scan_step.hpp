// The selective state space scan's single step: every env's states go through once.
#pragma once
#include "scan.hpp"

namespace mo {

// A channel's states lie over `lanes` neighbouring lanes (a power of two), V of them each, so that accesses run over the states as they lie; what
// is the channel's own is computed by each of its lanes. A workgroup has channels of STEP_ENVS envs, whose states it has in flight together, with the
// same decays; where an env's rows begin is computed once for all lanes. The states are all there is to move: 8 bytes each, which bound it.
// (32,768 envs, 512 channels of 16 states, bf16: 393 us, 5.8 TB/s; two envs a workgroup 456, eight 533; with every thread's own 64-bit offsets
// 581, a channel's states in one lane 3,300.)
// FAR: the states are more than the last-level cache holds, and go past it.
constexpr int STEP_ENVS = 4, STEP_THREADS = 256;
struct ScanStep {
    MoScan a;
    int lanes, log_lanes, blocks;    // workgroups of an env
};

// The sum over groups of `lanes` lanes, for all of them.
__device__ __forceinline__ float group_sum(float x, int lanes) {
    typedef unsigned U2 __attribute__((ext_vector_type(2)));
    if (lanes > 1) x += dpp<DPP_XOR1>(x);
    if (lanes > 2) x += dpp<DPP_XOR2>(x);
    if (lanes > 4) x += dpp<DPP_MIRROR8>(x);                  // (fours and eights hold one value each by now)
    if (lanes > 8) x += dpp<DPP_MIRROR16>(x);
    if (lanes > 16) {
        const U2 y = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
        x = __uint_as_float(y[0]) + __uint_as_float(y[1]);
    }
    if (lanes > 32) {
        const U2 y = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
        x = __uint_as_float(y[0]) + __uint_as_float(y[1]);
    }
    return x;
}

template <class T, int V, bool FAR> __global__ void __launch_bounds__(STEP_THREADS) k_scan_step(ScanStep k) {
    const MoScan& a = k.a;
    const int64_t block = block_here(), n0 = block / k.blocks * STEP_ENVS;
    if (n0 >= a.N) return;
    const unsigned id = (unsigned)(block % k.blocks) * blockDim.x + threadIdx.x, at = id >> k.log_lanes, q = id & (k.lanes - 1);
    const bool there = at < (unsigned)a.C, live = there && q * V < (unsigned)a.S;
    const unsigned c = there ? at : a.C - 1, s0 = live ? q * V : 0, g = a.G > 1 ? c / (a.C / a.G) : 0;    // (others read what there is)
    typedef Pack<float, V> P;
    typedef Pack<T, V> R;
    P h[STEP_ENVS];
    bool cut[STEP_ENVS];
    T x[STEP_ENVS], dt[STEP_ENVS], z[STEP_ENVS];
    R B[STEP_ENVS], C[STEP_ENVS];
    const int64_t env = (int64_t)a.C * a.S;
    const unsigned own = (c * a.S + s0) * 4;                  // (C <= 2^20, S <= 64: 2^28 bytes)
    const auto env_of = [&](int e) { return min(n0 + e, a.N - 1); };
#pragma unroll
    for (int e = 0; e < STEP_ENVS; e++) {
        const int64_t n = env_of(e);
        const auto row = [&](const MoRows& r) { return *lane_at((const T*)r.p + n * r.sn, c * (uint32_t)sizeof(T)); };
        const auto states = [&](const MoRows& r) { return *(const R*)((const T*)r.p + n * r.sn + g * r.sh + s0); };
        const P* p = lane_at((const P*)(a.state_out + n * env), own);
        h[e] = FAR ? streamed(p) : *p;
        cut[e] = a.start && a.start[n];
        x[e] = row(a.x);
        dt[e] = row(a.dt);
        if (a.z.p) z[e] = row(a.z);
        B[e] = states(a.Bt);
        C[e] = states(a.Ct);
    }
    const P A = *lane_at((const P*)a.A, own);
    const float bias = a.dt_bias ? a.dt_bias[c] : 0.f, D = a.D ? a.D[c] : 0.f;
#pragma unroll
    for (int e = 0; e < STEP_ENVS; e++) {
        if (n0 + e >= a.N) break;
        const float d = softplus(as_f32(dt[e]) + bias).d, u = d * as_f32(x[e]);
        float y = 0.f;
#pragma unroll
        for (int v = 0; v < V; v++) {
            const float add = u * as_f32(B[e].v[v]);
            h[e].v[v] = cut[e] ? add : fmaf(exp2_raw(d * (A.v[v] * LOG2E)), h[e].v[v], add);
            y = fmaf(as_f32(C[e].v[v]), h[e].v[v], y);
        }
        if (live) {
            P* p = lane_at((P*)(a.state_out + (n0 + e) * env), own);
            if (FAR) stream(p, h[e]);
            else *p = h[e];
        }
        y = group_sum(live ? y : 0.f, k.lanes);
        y = fmaf(D, a.D ? as_f32(x[e]) : 0.f, y);
        if (a.z.p) {
            const float zf = as_f32(z[e]);
            y *= zf * sigmoid(zf);
        }
        if (there && q == 0) *lane_at((T*)a.out.p + (n0 + e) * a.out.sn, c * (uint32_t)sizeof(T)) = as<T>(y);
    }
}

template <class T> int scan_step(const MoScan& a, hipStream_t s) {
    const auto fours = [](const MoRows& r) { return (uintptr_t)r.p % (4 * sizeof(T)) == 0 && r.sn % 4 == 0 && r.sh % 4 == 0; };
    const bool wide = a.S % 4 == 0 && (uintptr_t)a.state_out % 16 == 0 && (uintptr_t)a.A % 16 == 0 && fours(a.Bt) && fours(a.Ct);
    ScanStep k{a, 1, 0, 1};
    while (k.lanes * (wide ? 4 : 1) < a.S) k.lanes *= 2, k.log_lanes++;
    const int64_t lanes = (int64_t)a.C * k.lanes;
    const unsigned threads = (unsigned)std::min<int64_t>(STEP_THREADS, (lanes + kWave - 1) / kWave * kWave);
    k.blocks = (int)((lanes + threads - 1) / threads);
    const dim3 grid = grid_of((a.N + STEP_ENVS - 1) / STEP_ENVS * k.blocks), block(threads);
    const bool far = a.N * a.C * a.S * 4 > LAST_LEVEL_CACHE;
    if (wide && far) hipLaunchKernelGGL((k_scan_step<T, 4, true>), grid, block, 0, s, k);
    else if (wide) hipLaunchKernelGGL((k_scan_step<T, 4, false>), grid, block, 0, s, k);
    else hipLaunchKernelGGL((k_scan_step<T, 1, false>), grid, block, 0, s, k);
    return launched("k_scan_step");
}

}  // namespace mo
