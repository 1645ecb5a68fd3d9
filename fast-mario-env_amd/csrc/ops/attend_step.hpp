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
// lanes span the columns, and the 64 / CG lane groups take neighbouring rows, so that an access covers whole rows one after
// another; q and k go to the lanes through LDS, and the groups' sums of o are joined by shuffles. The state is all there is to
// move: 8 D E bytes, which bound it. (32,768 envs, 8 heads of 64, bf16: 1,440 us, 6.0 TB/s; with a lane's rows together instead of an access's, and
// q and k straight from memory, 2,310 us.)
// FAR: the states are more than the last-level cache holds, and go past it (1,523 us without); where they fit, the next step finds
// them there (2,000 envs: 83 us, 93 going past it).
template <class T, int V, int CG, bool FAR>
__global__ void __launch_bounds__(256) k_step_state(Step a) {
    constexpr int RG = kWave / CG, WAVES = 256 / kWave;
    __shared__ float sq[WAVES][MO_MAX_HEAD], sk[WAVES][MO_MAX_HEAD];
    const int lane = threadIdx.x % kWave, w = threadIdx.x / kWave, cg = lane % CG, rg = lane / CG;
    const int64_t nh = block_here() * WAVES + w;
    if (nh >= a.N * a.H) return;
    const int64_t n = nh / a.H;
    const int h = (int)(nh % a.H), e = (blockIdx.y * CG + cg) * V;
    const bool live = e < a.E;
    const auto at = [&](const MoRows& r) { return (T*)r.p + n * r.sn + h * r.sh; };
    const T *q = at(a.q), *k = at(a.k), *v = at(a.v);
    const bool cut = a.start && a.start[n];
    const float g = a.decay[h];
    typedef Pack<float, V> P;
    float* S = a.state + nh * (int64_t)a.D * a.E + e;
    P x[STEP_ROWS];
    const auto load = [&](int d0) {
#pragma unroll
        for (int r = 0; r < STEP_ROWS; r++) {
            const int d = d0 + r * RG + rg;
            if (d < a.D && live && !cut) {
                const P* p = (const P*)(S + (int64_t)d * a.E);
                x[r] = FAR ? streamed(p) : *p;
            }
        }
    };
    load(0);
    for (int d = lane; d < a.D; d += kWave) {
        sq[w][d] = as_f32(q[d]);
        sk[w][d] = as_f32(k[d]);
    }
    float vv[V], o[V];
#pragma unroll
    for (int c = 0; c < V; c++) { vv[c] = live ? as_f32(v[e + c]) : 0.f; o[c] = 0.f; }
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");     // (other lanes read them; a barrier alone orders no memory)
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
    for (int d0 = 0; d0 < a.D; d0 += STEP_ROWS * RG) {
        if (d0) load(d0);
#pragma unroll
        for (int r = 0; r < STEP_ROWS; r++) {
            const int d = d0 + r * RG + rg;
            if (d >= a.D || !live) continue;
            const float qd = sq[w][d], kd = sk[w][d];
#pragma unroll
            for (int c = 0; c < V; c++) {
                x[r].v[c] = cut ? kd * vv[c] : fmaf(g, x[r].v[c], kd * vv[c]);
                o[c] = fmaf(qd, x[r].v[c], o[c]);
            }
            P* p = (P*)(S + (int64_t)d * a.E);
            if (FAR) stream(p, x[r]);
            else *p = x[r];
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

// Four columns a lane where the state's rows allow 16-byte accesses, else one (and two launch rows where 64 lanes do not span them).
template <class T, bool FAR> int step_by_width(const Step& a, hipStream_t s) {
    const int64_t blocks = (a.N * a.H + 256 / kWave - 1) / (256 / kWave);
    const bool wide = a.E % 4 == 0 && (uintptr_t)a.state % 16 == 0;
    if (wide && a.E <= 32) hipLaunchKernelGGL((k_step_state<T, 4, 8, FAR>), grid_of(blocks), dim3(256), 0, s, a);
    else if (wide && a.E <= 64) hipLaunchKernelGGL((k_step_state<T, 4, 16, FAR>), grid_of(blocks), dim3(256), 0, s, a);
    else if (wide) hipLaunchKernelGGL((k_step_state<T, 4, 32, FAR>), grid_of(blocks), dim3(256), 0, s, a);
    else hipLaunchKernelGGL((k_step_state<T, 1, 64, FAR>), grid_of(blocks, (a.E + 63) / 64), dim3(256), 0, s, a);
    return launched("k_step_state");
}
template <class T> int step(const Step& a, hipStream_t s) {
    return a.N * a.H * a.D * a.E * 4 > LAST_LEVEL_CACHE ? step_by_width<T, true>(a, s) : step_by_width<T, false>(a, s);
}

}  // namespace mo
