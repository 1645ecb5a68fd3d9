// Linear attention's single step: the state of every env and head goes through once.
#pragma once
#include "common.hpp"

namespace mo {

struct Step {
    MoRows q, k, v, out;
    const float* decay;
    const uint8_t* start;
    float* state;
    int64_t N;
    int H, D, E;
    float scale;
};

constexpr int STEP_ROWS = 16;   // rows of the state that a lane has in flight

// S = (start ? 0 : g S) + k v^T and o = scale S^T q of one env and head in one wave. A lane holds V neighbouring columns, CG
// lanes span the columns, and the 64 / CG lane groups take D / (64 / CG) consecutive rows each, so a lane's q and k lie
// together; the groups' sums of o are joined by shuffles. The state is all there is to move: 8 D E bytes.
template <class T, int V, int CG>
__global__ void __launch_bounds__(256) k_step_state(Step a) {
    constexpr int RG = kWave / CG;
    const int lane = threadIdx.x % kWave, cg = lane % CG, rg = lane / CG;
    const int64_t nh = (int64_t)blockIdx.x * (256 / kWave) + threadIdx.x / kWave;
    if (nh >= a.N * a.H) return;
    const int64_t n = nh / a.H;
    const int h = (int)(nh % a.H), e = (blockIdx.y * CG + cg) * V;
    const bool live = e < a.E;
    const auto at = [&](const MoRows& r) { return (T*)r.p + n * r.sn + h * r.sh; };
    const T *q = at(a.q), *k = at(a.k), *v = at(a.v);
    const bool cut = a.start && a.start[n];
    const float g = a.decay[h];
    typedef Pack<float, V> P;
    float* S = a.state + nh * (int64_t)a.D * a.E;
    float vv[V], o[V];
#pragma unroll
    for (int c = 0; c < V; c++) { vv[c] = live ? as_f32(v[e + c]) : 0.f; o[c] = 0.f; }
    const int rows = (a.D + RG - 1) / RG, d1 = min(a.D, (rg + 1) * rows);
    for (int d0 = rg * rows; d0 < d1; d0 += STEP_ROWS) {
        P x[STEP_ROWS];
        float qq[STEP_ROWS], kk[STEP_ROWS];
#pragma unroll
        for (int r = 0; r < STEP_ROWS; r++) {
            const bool in = d0 + r < d1;
            if (in && live && !cut) x[r] = *(const P*)(S + (int64_t)(d0 + r) * a.E + e);
            qq[r] = in ? as_f32(q[d0 + r]) : 0.f;
            kk[r] = in ? as_f32(k[d0 + r]) : 0.f;
        }
#pragma unroll
        for (int r = 0; r < STEP_ROWS; r++) {
            if (d0 + r >= d1 || !live) continue;
#pragma unroll
            for (int c = 0; c < V; c++) {
                x[r].v[c] = cut ? kk[r] * vv[c] : fmaf(g, x[r].v[c], kk[r] * vv[c]);
                o[c] = fmaf(qq[r], x[r].v[c], o[c]);
            }
            stream((P*)(S + (int64_t)(d0 + r) * a.E + e), x[r]);
        }
    }
#pragma unroll
    for (int c = 0; c < V; c++)
        for (int m = CG; m < kWave; m *= 2) o[c] += __shfl_xor(o[c], m);
    if (rg == 0 && live) {
        T* y = at(a.out) + e;
#pragma unroll
        for (int c = 0; c < V; c++) y[c] = as<T>(o[c] * a.scale);
    }
}

// Four columns a lane where the state's rows allow 16-byte accesses, else one (and two lanes' worth of columns a launch row).
template <class T> int step(const Step& a, hipStream_t s) {
    const unsigned blocks = (unsigned)((a.N * a.H + 256 / kWave - 1) / (256 / kWave));
    const bool wide = a.E % 4 == 0 && (uintptr_t)a.state % 16 == 0;
    if (wide && a.E <= 32) hipLaunchKernelGGL((k_step_state<T, 4, 8>), dim3(blocks), dim3(256), 0, s, a);
    else if (wide && a.E <= 64) hipLaunchKernelGGL((k_step_state<T, 4, 16>), dim3(blocks), dim3(256), 0, s, a);
    else if (wide) hipLaunchKernelGGL((k_step_state<T, 4, 32>), dim3(blocks), dim3(256), 0, s, a);
    else hipLaunchKernelGGL((k_step_state<T, 1, 64>), dim3(blocks, (unsigned)((a.E + 63) / 64)), dim3(256), 0, s, a);
    return launched("k_step_state");
}

}  // namespace mo
