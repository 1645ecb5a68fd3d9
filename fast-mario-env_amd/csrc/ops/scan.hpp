// The selective state space scan over the steps of a rollout.
#pragma once
#include "sums.hpp"

namespace mo {

// A wave has 64 channels of one env, a lane all of a channel's states (or SP of them: then up to four waves share the channels and join their
// sums in LDS). B and C are the same for all lanes: they lie packed in float32 (k_scan_pack) and come as scalar loads, so a step of a
// state is one exponential, two products and two fused multiply-adds on registers.
constexpr int SCAN_STEPS = 8;        // steps of a chunk: between two kept states
constexpr int SCAN_WAVES = 4;
constexpr float LOG2E = 1.44269504088896340736f, LN2 = 0.69314718055994530942f;

struct Scan {
    MoScan a;
    const float* bc;                 // (T, N, G, 2, SB): B and C padded with zeros to whole slices
    float* kept;                     // (chunks, N, SB, C): the states before each chunk, for the gradient; or null
    float *seg_h, *seg_d;            // (segments, N, SB, C), (segments, N, C): see k_scan_enter
    float *part_bc, *part;           // (gradient) (per, T, N, G, 2, SB), (rows, SB + 2, C)
    int64_t chunks, each, segments;  // chunks of all steps, and of a segment
    int64_t rows;                    // (gradient) envs' segments that are taken at a time
    int slices, SB, Cg, per;         // waves that share channels, states padded, channels of a group, waves that span them
};

typedef const float __attribute__((address_space(4))) * Uniform;   // read by scalar loads: the same for all lanes, not written meanwhile
__device__ __forceinline__ Uniform uniform(const float* p) { return (Uniform)(uintptr_t)p; }

__device__ __forceinline__ float exp2_raw(float x) { return __builtin_amdgcn_exp2f(x); }
// softplus(r) = max(r, 0) + log1p(e), e = exp(-|r|) <= 1, by log1p(e) = 2 atanh(q), q = e / (2 + e) <= 1/3: the series to q^13 leaves 2e-8 of it.
struct Size { float d, slope; };     // and its derivative, 1 / (1 + exp(-r))
__device__ __forceinline__ Size softplus(float r) {
    const float e = exp2_raw(-fabsf(r) * LOG2E), q = e * __builtin_amdgcn_rcpf(2.f + e), q2 = q * q;
    float s = 2.f / 13.f;
    s = fmaf(s, q2, 2.f / 11.f);
    s = fmaf(s, q2, 2.f / 9.f);
    s = fmaf(s, q2, 2.f / 7.f);
    s = fmaf(s, q2, 2.f / 5.f);
    s = fmaf(s, q2, 2.f / 3.f);
    s = fmaf(s * q2, q, 2.f * q);
    return {fmaxf(r, 0.f) + s, (r < 0.f ? e : 1.f) * __builtin_amdgcn_rcpf(1.f + e)};
}
__device__ __forceinline__ float sigmoid(float z) { return __builtin_amdgcn_rcpf(1.f + exp2_raw(-z * LOG2E)); }

// B and C of every step in float32, padded.
template <class T> __global__ void __launch_bounds__(256) k_scan_pack(Scan k, float* bc) {
    const MoScan& a = k.a;
    const int64_t id = block_here() * 256 + threadIdx.x, row = id / (2 * k.SB);
    if (row >= a.T * a.N * a.G) return;
    const int i = (int)(id % (2 * k.SB)), s = i % k.SB, g = (int)(row % a.G);
    const int64_t n = row / a.G % a.N, t = row / a.G / a.N;
    const MoRows& r = i < k.SB ? a.Bt : a.Ct;
    bc[id] = s < a.S ? as_f32(((const T*)r.p)[t * r.st + n * r.sn + g * r.sh + s]) : 0.f;
}

// What a wave works on.
struct ScanPlace {
    int64_t n, segment;
    int g, c, lane, s0;              // group, this lane's channel, its first state
    bool live;
    __device__ __forceinline__ ScanPlace(const Scan& k, int64_t wave, int slice, int SP) {
        const int cbs = k.a.G * k.per, cb = (int)(wave % cbs);
        const int64_t rest = wave / cbs;
        n = rest % k.a.N;
        segment = rest / k.a.N;
        g = cb / k.per;
        lane = threadIdx.x % kWave;
        const int i = cb % k.per * kWave + lane;
        live = i < k.Cg;
        c = g * k.Cg + (live ? i : k.Cg - 1);
        s0 = slice * SP;
    }
};
__device__ __forceinline__ int wave_here() { return __builtin_amdgcn_readfirstlane(threadIdx.x / kWave); }

template <class T> __device__ __forceinline__ float at_row(const MoRows& r, int64_t t, int64_t n, int c) {
    return as_f32(((const T*)r.p)[t * r.st + n * r.sn + c]);
}
template <class T> __device__ __forceinline__ void to_row(const MoRows& r, int64_t t, int64_t n, int c, float x) {
    ((T*)r.p)[t * r.st + n * r.sn + c] = as<T>(x);
}
// Which of the SCAN_STEPS steps from t0 start an episode, as bits.
__device__ __forceinline__ unsigned starts_from(const MoScan& a, int64_t t0, int steps, int64_t n, int lane) {
    if (!a.start) return 0;
    return (unsigned)__ballot(lane < steps && a.start[(t0 + lane) * a.N + n]);
}
template <int SP> __device__ __forceinline__ void load_decays(const MoScan& a, int c, int s0, float (&A)[SP]) {
#pragma unroll
    for (int s = 0; s < SP; s++) A[s] = s0 + s < a.S ? a.A[(int64_t)c * a.S + s0 + s] * LOG2E : 0.f;
}

// Forward. SUMS: only what a segment adds to an entering state: its last states from zero, and the sum of its step sizes (-1 where an episode
// starts in it: nothing of what enters is left).
template <class T, int SP, bool SPLIT, bool SUMS>
__global__ void __launch_bounds__(SCAN_WAVES* kWave) k_scan(Scan k) {
    const MoScan& a = k.a;
    __shared__ float part[SPLIT ? SCAN_WAVES : 1][SCAN_STEPS][kWave];
    const int w = wave_here(), slice = SPLIT ? w : 0;
    const int64_t wave = SPLIT ? block_here() : block_here() * SCAN_WAVES + w;
    if (wave >= k.segments * a.N * a.G * k.per) return;
    const ScanPlace me(k, wave, slice, SP);
    const int64_t n = me.n, first = me.segment * k.each, last = min(k.chunks, first + k.each);
    const int c = me.c;
    float A[SP], h[SP], total = 0.f;
    load_decays<SP>(a, c, me.s0, A);
    const int64_t seg0 = ((me.segment * a.N + n) * k.SB + me.s0) * a.C + c;
#pragma unroll
    for (int s = 0; s < SP; s++) {
        if (SUMS) h[s] = 0.f;
        else if (k.segments > 1) h[s] = k.seg_h[seg0 + (int64_t)s * a.C];
        else h[s] = a.state && me.s0 + s < a.S ? a.state[(n * a.C + c) * a.S + me.s0 + s] : 0.f;
    }
    const float bias = a.dt_bias ? a.dt_bias[c] : 0.f, D = a.D ? a.D[c] : 0.f;
    const auto finish = [&](int64_t t, float y) {
        y = fmaf(D, a.D ? at_row<T>(a.x, t, n, c) : 0.f, y);
        if (a.z.p) {
            const float z = at_row<T>(a.z, t, n, c);
            y *= z * sigmoid(z);
        }
        if (me.live) to_row<T>(a.out, t, n, c, y);
    };
    for (int64_t chunk = first; chunk < last; chunk++) {
        const int64_t t0 = chunk * SCAN_STEPS;
        const int steps = (int)min((int64_t)SCAN_STEPS, a.T - t0);
        const unsigned cuts = starts_from(a, t0, steps, n, me.lane);
        if (!SUMS && k.kept && me.live) {
            float* to = k.kept + ((chunk * a.N + n) * k.SB + me.s0) * a.C + c;
#pragma unroll
            for (int s = 0; s < SP; s++) to[(int64_t)s * a.C] = h[s];
        }
#pragma unroll
        for (int i = 0; i < SCAN_STEPS; i++) {
            if (i >= steps) break;
            const int64_t t = t0 + i;
            const float x = at_row<T>(a.x, t, n, c), d = softplus(at_row<T>(a.dt, t, n, c) + bias).d, u = d * x;
            const Uniform B = uniform(k.bc + ((t * a.N + n) * a.G + me.g) * 2 * k.SB + me.s0), C = B + k.SB;
            if (cuts >> i & 1) {
#pragma unroll
                for (int s = 0; s < SP; s++) h[s] = 0.f;
                total = -1.f;
            }
            if (SUMS && total >= 0.f) total += d;
            float y = 0.f;
#pragma unroll
            for (int s = 0; s < SP; s++) {
                h[s] = fmaf(exp2_raw(d * A[s]), h[s], u * B[s]);
                if (!SUMS) y = fmaf(C[s], h[s], y);
            }
            if (SUMS) continue;
            if (SPLIT) part[slice][i][me.lane] = y;
            else finish(t, y);
        }
        if (SPLIT && !SUMS) {
            __syncthreads();
            for (int i = slice; i < steps; i += k.slices) {
                float y = 0.f;
                for (int s = 0; s < k.slices; s++) y += part[s][i][me.lane];
                finish(t0 + i, y);
            }
            __syncthreads();
        }
    }
    if (!me.live) return;
    if (SUMS) {
#pragma unroll
        for (int s = 0; s < SP; s++) k.seg_h[seg0 + (int64_t)s * a.C] = h[s];
        if (slice == 0) k.seg_d[(me.segment * a.N + n) * a.C + c] = total;
    } else if (last == k.chunks) {
#pragma unroll
        for (int s = 0; s < SP; s++)
            if (me.s0 + s < a.S) a.state_out[(n * a.C + c) * a.S + me.s0 + s] = h[s];
    }
}

// From what each segment adds to what enters each (in place): forwards in time from the state, or (BACK) backwards from its gradient.
template <bool BACK> __global__ void __launch_bounds__(256) k_scan_enter(Scan k) {
    const MoScan& a = k.a;
    const int64_t id = block_here() * 256 + threadIdx.x, row = id / a.C;
    if (row >= a.N * k.SB) return;
    const int c = (int)(id % a.C), s = (int)(row % k.SB);
    const int64_t n = row / k.SB;
    const bool real = s < a.S;
    const float* from = BACK ? a.dstate_out : a.state;
    const float A = real ? a.A[(int64_t)c * a.S + s] * LOG2E : 0.f;
    float h = from && real ? from[(n * a.C + c) * a.S + s] : 0.f;
    for (int64_t i = 0; i < k.segments; i++) {
        const int64_t j = BACK ? k.segments - 1 - i : i;
        float* at = k.seg_h + ((j * a.N + n) * k.SB + s) * a.C + c;
        const float d = k.seg_d[(j * a.N + n) * a.C + c], add = *at;
        *at = h;
        h = d < 0.f ? add : fmaf(exp2_raw(d * A), h, add);
    }
}

// ---- host side
struct ScanCut { int SP, slices; };
inline ScanCut scan_slices(int S) {
    const int slices = (S + 15) / 16, SP = ((S + slices - 1) / slices + 3) / 4 * 4;
    return {SP, slices};
}
constexpr int64_t SCAN_FILL = 4096;     // waves that fill the card
inline Scan scan_cut(const MoScan& a, bool backward) {
    Scan k{};
    k.a = a;
    const ScanCut c = scan_slices(a.S);
    k.slices = c.slices;
    k.SB = c.SP * c.slices;
    k.Cg = a.C / a.G;
    k.per = (k.Cg + kWave - 1) / kWave;
    k.chunks = (a.T + SCAN_STEPS - 1) / SCAN_STEPS;
    // Few sequences are cut over their length: each segment is gone through twice, once for what it adds to the state.
    const int64_t waves = std::max<int64_t>(1, a.N * a.G * k.per * k.slices), most = std::max<int64_t>(1, SCAN_FILL / waves);
    k.segments = most >= 4 ? std::min(most, std::max<int64_t>(1, k.chunks / 4)) : 1;
    k.each = std::max<int64_t>(1, (k.chunks + k.segments - 1) / k.segments);
    k.segments = std::max<int64_t>(1, (k.chunks + k.each - 1) / k.each);
    k.rows = backward ? std::min(k.segments * a.N, std::max<int64_t>(1, 2 * SCAN_FILL / (a.G * k.per * k.slices))) : 0;
    return k;
}
// In floats, each part a multiple of 4 of them.
inline int64_t whole(int64_t n) { return (n + 3) / 4 * 4; }
inline int64_t scan_bc(const Scan& k) { return whole(k.a.T * k.a.N * k.a.G * 2 * k.SB); }
inline int64_t scan_kept(const Scan& k) { return whole(k.chunks * k.a.N * k.SB * k.a.C); }
inline int64_t scan_segs(const Scan& k) { return k.segments > 1 ? whole(k.segments * k.a.N * (k.SB + 1) * k.a.C) : 0; }
inline int64_t scan_parts_bc(const Scan& k) { return whole(k.per * k.a.T * k.a.N * k.a.G * 2 * k.SB); }
inline int64_t scan_parts(const Scan& k) { return whole(k.rows * (k.SB + 2) * k.a.C); }
inline int64_t scan_work_floats(const Scan& k, bool backward) {
    if (!backward) return (k.a.saved ? 0 : scan_bc(k)) + scan_segs(k);
    return scan_segs(k) + scan_parts_bc(k) + scan_parts(k) + column_sums_work(k.rows, k.SB + 2, k.a.C);
}

template <class F> int by_states(const Scan& k, F f) {
    const int SP = k.SB / k.slices;
    if (k.slices == 1) {
        if (SP == 4) return f(std::integral_constant<int, 4>{}, std::false_type{});
        if (SP == 8) return f(std::integral_constant<int, 8>{}, std::false_type{});
        if (SP == 12) return f(std::integral_constant<int, 12>{}, std::false_type{});
        return f(std::integral_constant<int, 16>{}, std::false_type{});
    }
    if (SP == 12) return f(std::integral_constant<int, 12>{}, std::true_type{});
    return f(std::integral_constant<int, 16>{}, std::true_type{});
}
inline void scan_launch_shape(const Scan& k, int64_t waves, dim3& grid, dim3& block) {
    grid = grid_of(k.slices > 1 ? waves : (waves + SCAN_WAVES - 1) / SCAN_WAVES);
    block = dim3(kWave * (k.slices > 1 ? k.slices : SCAN_WAVES));
}

template <class T> int scan_forward(const MoScan& a, hipStream_t s) {
    Scan k = scan_cut(a, false);
    float* bc = (float*)(a.saved ? a.saved : a.work);
    k.bc = bc;
    k.kept = a.saved ? bc + scan_bc(k) : nullptr;
    k.seg_h = (float*)a.work + (a.saved ? 0 : scan_bc(k));
    k.seg_d = k.seg_h + k.segments * a.N * k.SB * a.C;
    if (a.T) {
        const int64_t n = a.T * a.N * a.G * 2 * k.SB;
        hipLaunchKernelGGL((k_scan_pack<T>), grid_of((n + 255) / 256), dim3(256), 0, s, k, bc);
        if (launched("k_scan_pack")) return -1;
    }
    return by_states(k, [&](auto sp, auto split) {
        constexpr int SP = decltype(sp)::value;
        constexpr bool SPLIT = decltype(split)::value;
        dim3 grid, block;
        scan_launch_shape(k, k.segments * a.N * a.G * k.per, grid, block);
        if (k.segments > 1) {
            hipLaunchKernelGGL((k_scan<T, SP, SPLIT, true>), grid, block, 0, s, k);
            hipLaunchKernelGGL((k_scan_enter<false>), grid_of((a.N * k.SB * a.C + 255) / 256), dim3(256), 0, s, k);
        }
        hipLaunchKernelGGL((k_scan<T, SP, SPLIT, false>), grid, block, 0, s, k);
        return launched("k_scan");
    });
}

}  // namespace mo
