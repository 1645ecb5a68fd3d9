// Group norm with an activation where a sample fits a workgroup's registers: read once.
#pragma once
#include "norm_general.hpp"

namespace mo {

// A team of threads (W waves, or of a small sample a part of one) takes a sample, holds it as up to R packs of 8 channels a thread
// and goes on to its next sample. A thread has the packs cv = t % NV (NV: packs a pixel, rounded up to a power of two; threads of
// packs that are not there idle) of the pixels t / NV, t / NV + TT / NV, .. (TT: the team's threads), so its channels, their weights
// and their gradients' sums stay its own. Sums over a group are shuffles over the lanes that hold it, and one exchange through LDS
// where the team has several waves (MULTI). The mean's sum goes about the group's first value, and the variance is that of the
// values in registers about their mean: a large mean costs neither digits, and equal values have no deviations. NS: groups of a pack, each with sums of its own: 1 (a group is whole packs), 2, 4 or 8.
// Bound by memory, a value read and one written (back: two and one). Measured, bf16, in microseconds: 4,096 x 32 x 20 x 20 in 4 groups 38
// (5.6 TB/s, partly out of the last-level cache), 104 through norm_general; 262,144 x 512 in 8 groups 120 (4.5 TB/s), with the gradient 275; 4,096 x
// 64 x 9 x 9 in 8 groups forward 21, back 33; groups of one channel need eight sums a pack and more registers: 16,384 x 32 x 9 x 9
// forward and back 216 in 32 groups, 105 in 8, 95 in 4. (LDS by the team's waves: room for eight waves in each block made the 216 340.) The
// gradients of four bf16 packs a thread in groups of 4 channels keep 4 to 6 registers in scratch.
struct Small {
    MoNorm a;
    int W, TT, nv, NV, log_nv; // waves and threads a team; packs a pixel, and rounded up
    int cg, vpg;               // channels a group; packs a group (at least 1)
    bool far;                  // rows (R = 1) of an x that fills the last-level cache come past it (262,144 x 512 bf16: gradient 186 ->
                               // 176 us); a smaller x may be there from its maker, and larger samples gain nothing
    float* part;               // (blocks, 2, C): the blocks' sums for dweight and dbias
};

constexpr int SMALL_PACKS = 8, SMALL_PACKS_BACK = 4;   // packs a thread, at most
constexpr int SMALL_WAVES = 8;                          // waves a team, at most
constexpr int small_threads(bool multi) { return multi ? SMALL_WAVES * kWave : 256; }   // (one wave a sample: four samples a block)

// The sums over a group's lanes, pixels and waves of a thread's NS values; x: a set for each of two exchanges in turn, so that
// one barrier a sum is enough.
template <bool MULTI, int NS, int SETS>
__device__ __forceinline__ void group_sum(float (&s)[NS], const Small& k, float (*x)[kWave][NS], int turn) {
    const int lane = threadIdx.x % kWave;
#pragma unroll
    for (int i = 0; i < NS; i++)
        for (int m = k.NV; m < (MULTI ? kWave : k.TT); m *= 2) s[i] += __shfl_xor(s[i], m);
    if (NS == SETS) {                                      // whole packs: a value a set
        if ((k.vpg & (k.vpg - 1)) == 0) {
#pragma unroll
            for (int i = 0; i < NS; i++)
                for (int m = 1; m < k.vpg; m *= 2) s[i] += __shfl_xor(s[i], m);
        } else {
            const int cv = lane & (k.NV - 1), first = lane - cv + cv / k.vpg * k.vpg;
#pragma unroll
            for (int i = 0; i < NS; i++) {
                float t = 0.f;
                for (int j = 0; j < k.vpg; j++) t += __shfl(s[i], first + j);
                s[i] = t;
            }
        }
    }
    if (!MULTI) return;
    x += turn * k.W;
#pragma unroll
    for (int i = 0; i < NS; i++) x[threadIdx.x / kWave][lane][i] = s[i];
    __syncthreads();
#pragma unroll
    for (int i = 0; i < NS; i++) s[i] = 0.f;
    for (int j = 0; j < k.W; j++)
#pragma unroll
        for (int i = 0; i < NS; i++) s[i] += x[j][lane][i];
}

extern __shared__ __align__(16) float small_lds[];       // MULTI: two exchanges by wave; going back, then the waves' sums for dweight
inline unsigned small_lds_bytes(bool multi, int waves, int NS, bool backward) {
    const int exchange = multi ? 2 * waves * kWave * NS * (backward ? 2 : 1) : 0;
    return 4 * (unsigned)std::max(exchange, backward ? waves * kWave * 8 : 0);
}

template <class T, bool MULTI, int R, int ACT, int NS>
__global__ void __launch_bounds__(small_threads(MULTI)) k_norm_small(Small k) {
    constexpr int PER = 8 / NS;   // a pack's channels of one group
    typedef Pack<T, 8> P;
    float (*x)[kWave][NS] = (float (*)[kWave][NS])small_lds;
    const MoNorm& a = k.a;
    const int TT = k.TT, teams = MULTI ? 1 : 256 / TT;
    const int t = threadIdx.x & (TT - 1), cv = t & (k.NV - 1), pl = t >> k.log_nv, PL = TT >> k.log_nv, S = (int)a.S;
    const bool live = cv < k.nv;
    float w[8], s[8];
#pragma unroll
    for (int i = 0; i < 8; i++) {
        w[i] = live && a.weight ? a.weight[cv * 8 + i] : 1.f;
        s[i] = live && a.bias ? a.bias[cv * 8 + i] : 0.f;
    }
    const float n = (float)a.S * (float)k.cg, by = 1.f / n;
    const int first = cv - cv % k.vpg;                         // the pack that the thread's group begins in
    for (int64_t b = (int64_t)blockIdx.x * teams + (MULTI ? 0 : threadIdx.x / TT); b < a.B; b += (int64_t)gridDim.x * teams) {
        const T* in = (const T*)a.x + b * a.S * a.C + cv * 8;
        P v[R];
#pragma unroll
        for (int r = 0; r < R; r++)
            if (live && pl + r * PL < S) {
                const P* p = (const P*)(in + (int64_t)(pl + r * PL) * a.C);
                v[r] = R == 1 && k.far ? streamed(p) : *p;
            }
        float mean[NS] = {}, var[NS] = {}, x0[NS];             // x0: each group's first value, from the lane that holds it or from memory
#pragma unroll
        for (int i = 0; i < NS; i++)
            x0[i] = !MULTI ? __shfl(as_f32(v[0].v[i * PER]), (threadIdx.x & (kWave - TT)) + first)
                    : live ? as_f32(((const T*)a.x)[b * a.S * a.C + first * 8 + i * PER]) : 0.f;
#pragma unroll
        for (int r = 0; r < R; r++)
            if (live && pl + r * PL < S)
#pragma unroll
                for (int i = 0; i < 8; i++) mean[i / PER] += as_f32(v[r].v[i]) - x0[i / PER];
        group_sum<MULTI, NS, 1>(mean, k, x, 0);
#pragma unroll
        for (int i = 0; i < NS; i++) mean[i] = x0[i] + mean[i] / n;
#pragma unroll
        for (int r = 0; r < R; r++)
            if (live && pl + r * PL < S)
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    const float d = as_f32(v[r].v[i]) - mean[i / PER];
                    var[i / PER] = fmaf(d, d, var[i / PER]);
                }
        group_sum<MULTI, NS, 1>(var, k, x, 1);
        float rstd[NS];
#pragma unroll
        for (int i = 0; i < NS; i++) rstd[i] = 1.f / sqrtf(fmaf(var[i], by, a.eps));
        if (a.stats && pl == 0 && live)
#pragma unroll
            for (int i = 0; i < NS; i++)
                if ((cv * 8 + i * PER) % k.cg == 0) {
                    float* to = a.stats + 2 * (b * a.groups + (cv * 8 + i * PER) / k.cg);
                    to[0] = mean[i];
                    to[1] = rstd[i];
                }
        T* out = (T*)a.y + b * a.S * a.C + cv * 8;
#pragma unroll
        for (int r = 0; r < R; r++)
            if (live && pl + r * PL < S) {
#pragma unroll
                for (int i = 0; i < 8; i++)
                    v[r].v[i] = as<T>(act<ACT>(fmaf((as_f32(v[r].v[i]) - mean[i / PER]) * rstd[i / PER], w[i], s[i])));
                stream((P*)(out + (int64_t)(pl + r * PL) * a.C), v[r]);
            }
    }
}

template <class T, bool MULTI, int R, int ACT, int NS>
__global__ void __launch_bounds__(small_threads(MULTI), (NS <= 2 && sizeof(T) == 2 ? 4 : 2)) k_norm_small_back(Small k) {
    constexpr int PER = 8 / NS;   // a pack's channels of one group
    typedef Pack<T, 8> P;
    float (*x)[kWave][2 * NS] = (float (*)[kWave][2 * NS])small_lds, (*sums)[kWave][8] = (float (*)[kWave][8])small_lds;
    const MoNorm& a = k.a;
    const int TT = k.TT, teams = MULTI ? 1 : 256 / TT, waves = MULTI ? k.W : 4;
    const int t = threadIdx.x & (TT - 1), cv = t & (k.NV - 1), pl = t >> k.log_nv, PL = TT >> k.log_nv, S = (int)a.S;
    const bool live = cv < k.nv;
    float w[8], s[8], dw[8] = {}, db[8] = {};
#pragma unroll
    for (int i = 0; i < 8; i++) {
        w[i] = live && a.weight ? a.weight[cv * 8 + i] : 1.f;
        s[i] = live && a.bias ? a.bias[cv * 8 + i] : 0.f;
    }
    const float by = 1.f / ((float)a.S * (float)k.cg);
    int turn = 0;
    for (int64_t b = (int64_t)blockIdx.x * teams + (MULTI ? 0 : threadIdx.x / TT); b < a.B; b += (int64_t)gridDim.x * teams) {
        const int64_t at = b * a.S * a.C + cv * 8;
        P v[R], dy[R];
#pragma unroll
        for (int r = 0; r < R; r++)
            if (live && pl + r * PL < S) {
                const P *p = (const P*)((const T*)a.x + at + (int64_t)(pl + r * PL) * a.C), *d = (const P*)((const T*)a.dy + at + (int64_t)(pl + r * PL) * a.C);
                v[r] = R == 1 && k.far ? streamed(p) : *p;
                dy[r] = R == 1 && k.far ? streamed(d) : *d;
            }
        float mean[NS], rstd[NS], m[2 * NS] = {};          // m: the sums of dh, then those of dh h
#pragma unroll
        for (int i = 0; i < NS; i++) {
            const float* st = a.stats + 2 * (b * a.groups + (live ? (cv * 8 + i * PER) / k.cg : 0));
            mean[i] = st[0];
            rstd[i] = st[1];
        }
        float dh[R][8];
#pragma unroll
        for (int r = 0; r < R; r++)
            if (live && pl + r * PL < S)
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    const float h = (as_f32(v[r].v[i]) - mean[i / PER]) * rstd[i / PER];
                    const float dz = as_f32(dy[r].v[i]) * act_grad<ACT>(fmaf(h, w[i], s[i]));
                    dw[i] = fmaf(dz, h, dw[i]);
                    db[i] += dz;
                    dh[r][i] = dz * w[i];
                    m[i / PER] += dh[r][i];
                    m[NS + i / PER] = fmaf(dh[r][i], h, m[NS + i / PER]);
                }
        group_sum<MULTI, 2 * NS, 2>(m, k, x, turn);
        turn ^= 1;
#pragma unroll
        for (int i = 0; i < 2 * NS; i++) m[i] *= by;
#pragma unroll
        for (int r = 0; r < R; r++)
            if (live && pl + r * PL < S) {
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    const float h = (as_f32(v[r].v[i]) - mean[i / PER]) * rstd[i / PER];
                    v[r].v[i] = as<T>(rstd[i / PER] * (dh[r][i] - fmaf(h, m[NS + i / PER], m[i / PER])));
                }
                stream((P*)((T*)a.dx + at + (int64_t)(pl + r * PL) * a.C), v[r]);
            }
    }
    if (!k.part) return;
    // the block's sums for dweight and dbias: over the pixel lanes, then over its waves in order
#pragma unroll
    for (int i = 0; i < 8; i++)
        for (int m = k.NV; m < kWave; m *= 2) {
            dw[i] += __shfl_xor(dw[i], m);
            db[i] += __shfl_xor(db[i], m);
        }
    for (int half = 0; half < 2; half++) {
        __syncthreads();
        if (threadIdx.x % kWave < k.NV)
#pragma unroll
            for (int i = 0; i < 8; i++) sums[threadIdx.x / kWave][threadIdx.x % kWave][i] = half ? db[i] : dw[i];
        __syncthreads();
        for (int c = threadIdx.x; c < a.C; c += blockDim.x) {
            float sum = 0.f;
            for (int j = 0; j < waves; j++) sum += sums[j][c / 8][c % 8];
            k.part[((int64_t)blockIdx.x * 2 + half) * a.C + c] = sum;
        }
    }
}

// ---- host side
struct SmallCut { int W, TT, R, blocks; };

// Whole packs a pixel, groups of whole packs or of 1, 2 or 4 channels, a pixel's packs within a wave (64 packs, 512 channels: sums are
// shuffles of a wave, and waves exchange them lane by lane), and a sample within a team's registers. Wider pixels and other groups go to
// norm_rows, by single elements (65,536 x 1,024 in 8 groups, forward and gradient 429 us; its bytes take 129), and samples that fit neither
// go through memory twice (norm_general).
inline bool norm_small_takes(const MoNorm& a, bool backward, SmallCut& c) {
    const int cg = a.C / a.groups;
    if (!norm_wide(a) || a.C > 8 * kWave || (cg % 8 && 8 % cg)) return false;
    int NV = 1;
    while (NV < a.C / 8) NV *= 2;
    const int most = backward ? SMALL_PACKS_BACK : SMALL_PACKS;
    const int64_t packs = a.S * NV;
    if (packs > (int64_t)SMALL_WAVES * kWave * most) return false;
    for (c.W = 1; packs > (int64_t)c.W * kWave * most; c.W *= 2) {}
    for (c.R = 1; packs > (int64_t)c.W * kWave * c.R; c.R *= 2) {}
    for (c.TT = NV; c.TT < c.W * kWave && c.TT < packs; c.TT *= 2) {}
    const int per_block = c.W == 1 ? 256 / c.TT : 1, waves = c.W == 1 ? 4 : c.W;
    const int64_t blocks = (a.B + per_block - 1) / per_block, fill = (int64_t)compute_units() * std::max(1, (backward ? 16 : 32) / waves);
    c.blocks = (int)std::min(blocks, fill);
    return true;
}

template <class T, bool MULTI, int R, int ACT> int norm_small_run(const Small& k, const SmallCut& c, bool backward, hipStream_t s) {
    const dim3 block(MULTI ? c.W * kWave : 256);
    const auto go = [&](auto ns) {
        constexpr int NS = decltype(ns)::value;
        const unsigned lds = small_lds_bytes(MULTI, MULTI ? c.W : 4, NS, backward);
        if (!backward) hipLaunchKernelGGL((k_norm_small<T, MULTI, R, ACT, NS>), dim3(c.blocks), block, lds, s, k);
        else if constexpr (R <= SMALL_PACKS_BACK) hipLaunchKernelGGL((k_norm_small_back<T, MULTI, R, ACT, NS>), dim3(c.blocks), block, lds, s, k);
        return launched("k_norm_small");
    };
    return k.cg % 8 == 0 ? go(std::integral_constant<int, 1>{}) : k.cg == 4 ? go(std::integral_constant<int, 2>{})
         : k.cg == 2 ? go(std::integral_constant<int, 4>{}) : go(std::integral_constant<int, 8>{});
}

template <class T, int ACT> int norm_small(const MoNorm& a, const SmallCut& c, bool backward, hipStream_t s) {
    const int cg = a.C / a.groups;
    Small k{a, c.W, c.TT, a.C / 8, 1, 0, cg, std::max(1, cg / 8),
            a.B * a.S * a.C * (int64_t)sizeof(T) >= LAST_LEVEL_CACHE, nullptr};
    while (k.NV < k.nv) { k.NV *= 2; k.log_nv++; }
    if (backward && a.dweight) k.part = (float*)a.work;
    int rc;
    if (c.W == 1 && c.R == 1) rc = norm_small_run<T, false, 1, ACT>(k, c, backward, s);
    else if (c.W == 1 && c.R == 2) rc = norm_small_run<T, false, 2, ACT>(k, c, backward, s);
    else if (c.W == 1 && c.R == 4) rc = norm_small_run<T, false, 4, ACT>(k, c, backward, s);
    else if (c.W == 1) rc = norm_small_run<T, false, 8, ACT>(k, c, backward, s);
    else if (backward) rc = norm_small_run<T, true, 4, ACT>(k, c, backward, s);
    else rc = norm_small_run<T, true, 8, ACT>(k, c, backward, s);
    if (rc || !k.part) return rc;
    return norm_colsum(a, k.part, c.blocks, k.part + (int64_t)c.blocks * 2 * a.C, s);
}

inline int64_t norm_small_work(const MoNorm& a, const SmallCut& c, bool backward) {   // in floats
    return backward && a.dweight ? ((int64_t)c.blocks + NORM_SUM_ROWS) * 2 * a.C : 0;
}

}  // namespace mo
