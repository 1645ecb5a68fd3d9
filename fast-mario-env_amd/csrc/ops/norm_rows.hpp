// Group norm with an activation where a sample's group fits a wave's registers and norm_small does not take it: channels or groups that are
// not whole 16-byte packs, buffers off 16 bytes, and pixels of more than 512 channels. Read once, an element an access.
#pragma once
#include "norm_general.hpp"

namespace mo {

// A team of TT lanes (a power of two up to a wave) holds one group of one sample, up to R values a lane, and goes on to the same
// group of a later sample, so that a lane's channels, their weights and their gradients' sums stay its own. Lane l has channel
// l % cg of the pixels l / cg, l / cg + PL, ..; of a single pixel of more than 64 channels (ONE) the channels l, l + 64, ...
// Neighbouring teams have neighbouring groups, whose values lie together.
// Against norm_general's slabs (a block a sample, and one a group to join them), forward and gradient in microseconds: 200,000 x 30
// float32 in 5 groups 74 instead of 2,768, 8,192 x 96 x 3 x 3 bf16 in 16 groups 75 instead of 477, 65,536 x 1,024 bf16 in 8 groups 429
// instead of 3,163 (1.6 TB/s: two bytes a lane and access), 8,192 x 24 x 9 x 9 bf16 in 4 groups 158 instead of 218.
struct Rows {
    MoNorm a;
    int cg, TT, PL;
    int64_t rows;              // samples that are taken at a time: teams by group
    float* part;               // (rows, 2, C): each team's sums for dweight and dbias
};

constexpr int ROWS_MOST = 16;  // values a lane, at most

__device__ __forceinline__ float team_sum(float x, int TT) {
    for (int m = 1; m < TT; m *= 2) x += __shfl_xor(x, m);
    return x;
}

// Which group and samples a thread's team has, and where its values are.
template <bool ONE> struct Place {
    int l, c, p, g;
    int64_t b;
    bool live;
    __device__ __forceinline__ Place(const Rows& k) {
        const int64_t team = ((int64_t)blockIdx.x * NORM_THREADS + threadIdx.x) / k.TT;
        l = threadIdx.x & (k.TT - 1);
        c = ONE ? l : l % k.cg;
        p = ONE ? 0 : l / k.cg;
        g = (int)(team % k.a.groups);
        b = team / k.a.groups;                 // (past the last team: b >= rows)
        live = ONE || p < k.PL;
    }
    __device__ __forceinline__ bool has(const Rows& k, int r) const { return ONE ? c + r * kWave < k.cg : live && p + r * k.PL < (int)k.a.S; }
    __device__ __forceinline__ int channel(const Rows& k, int r) const { return g * k.cg + c + (ONE ? r * kWave : 0); }
    __device__ __forceinline__ int64_t at(const Rows& k, int64_t sample, int r) const {
        return (sample * k.a.S + (ONE ? 0 : p + r * k.PL)) * k.a.C + channel(k, r);
    }
};

template <class T, int R, bool ONE, int ACT>
__global__ void __launch_bounds__(NORM_THREADS) k_norm_rows(Rows k) {
    constexpr int K = ONE ? R : 1;
    const MoNorm& a = k.a;
    const Place<ONE> me(k);
    if (me.b >= k.rows) return;
    float w[K], s[K];
#pragma unroll
    for (int i = 0; i < K; i++) {
        const bool there = a.weight && me.has(k, i);
        w[i] = there ? a.weight[me.channel(k, i)] : 1.f;
        s[i] = there ? a.bias[me.channel(k, i)] : 0.f;
    }
    const float by = 1.f / ((float)a.S * (float)k.cg);
    for (int64_t b = me.b; b < a.B; b += k.rows) {
        float x[R], mean = 0.f, var = 0.f;
#pragma unroll
        for (int r = 0; r < R; r++) x[r] = me.has(k, r) ? as_f32(((const T*)a.x)[me.at(k, b, r)]) : 0.f;
        const float x0 = __shfl(x[0], threadIdx.x & (kWave - k.TT));   // sums go about the first value: a large mean costs no digits
#pragma unroll
        for (int r = 0; r < R; r++) mean += me.has(k, r) ? x[r] - x0 : 0.f;
        mean = team_sum(mean, k.TT) * by;
#pragma unroll
        for (int r = 0; r < R; r++) {
            x[r] = x[r] - x0 - mean;
            var = me.has(k, r) ? fmaf(x[r], x[r], var) : var;
        }
        const float rstd = 1.f / sqrtf(fmaf(team_sum(var, k.TT), by, a.eps));
        if (a.stats && me.l == 0) {
            a.stats[2 * (b * a.groups + me.g)] = x0 + mean;
            a.stats[2 * (b * a.groups + me.g) + 1] = rstd;
        }
#pragma unroll
        for (int r = 0; r < R; r++)
            if (me.has(k, r)) ((T*)a.y)[me.at(k, b, r)] = as<T>(act<ACT>(fmaf(x[r] * rstd, w[r % K], s[r % K])));
    }
}

template <class T, int R, bool ONE, int ACT>
__global__ void __launch_bounds__(NORM_THREADS) k_norm_rows_back(Rows k) {
    constexpr int K = ONE ? R : 1;
    __shared__ float lds[2][NORM_THREADS];
    const MoNorm& a = k.a;
    const Place<ONE> me(k);
    float w[K], s[K], dw[K] = {}, db[K] = {};
#pragma unroll
    for (int i = 0; i < K; i++) {
        const bool there = a.weight && me.has(k, i);
        w[i] = there ? a.weight[me.channel(k, i)] : 1.f;
        s[i] = there ? a.bias[me.channel(k, i)] : 0.f;
    }
    const float by = 1.f / ((float)a.S * (float)k.cg);
    for (int64_t b = me.b < k.rows ? me.b : a.B; b < a.B; b += k.rows) {
        const float* st = a.stats + 2 * (b * a.groups + me.g);
        const float mean = st[0], rstd = st[1];
        float h[R], dh[R], m1 = 0.f, m2 = 0.f;
#pragma unroll
        for (int r = 0; r < R; r++) {
            h[r] = me.has(k, r) ? as_f32(((const T*)a.x)[me.at(k, b, r)]) : mean;
            dh[r] = me.has(k, r) ? as_f32(((const T*)a.dy)[me.at(k, b, r)]) : 0.f;
        }
#pragma unroll
        for (int r = 0; r < R; r++)
            if (me.has(k, r)) {
                h[r] = (h[r] - mean) * rstd;
                const float dz = dh[r] * act_grad<ACT>(fmaf(h[r], w[r % K], s[r % K]));
                dw[r % K] = fmaf(dz, h[r], dw[r % K]);
                db[r % K] += dz;
                dh[r] = dz * w[r % K];
                m1 += dh[r];
                m2 = fmaf(dh[r], h[r], m2);
            }
        m1 = team_sum(m1, k.TT) * by;
        m2 = team_sum(m2, k.TT) * by;
#pragma unroll
        for (int r = 0; r < R; r++)
            if (me.has(k, r)) ((T*)a.dx)[me.at(k, b, r)] = as<T>(rstd * (dh[r] - fmaf(h[r], m2, m1)));
    }
    if (!k.part) return;
    float* to = k.part + me.b * 2 * a.C;
    if (ONE) {
#pragma unroll
        for (int r = 0; r < R; r++)
            if (me.b < k.rows && me.has(k, r)) {
                to[me.channel(k, r)] = dw[r % K];
                to[a.C + me.channel(k, r)] = db[r % K];
            }
        return;
    }
    lds[0][threadIdx.x] = dw[0];                       // a channel's sums over its pixel lanes, in order
    lds[1][threadIdx.x] = db[0];
    __syncthreads();
    if (me.b >= k.rows || me.l >= k.cg) return;
    float s1 = 0.f, s2 = 0.f;
    for (int p = 0; p < k.PL; p++) {
        s1 += lds[0][threadIdx.x + p * k.cg];
        s2 += lds[1][threadIdx.x + p * k.cg];
    }
    to[me.channel(k, 0)] = s1;
    to[a.C + me.channel(k, 0)] = s2;
}

// ---- host side
struct RowsCut { int TT, PL, R, blocks; bool one; int64_t rows; };

inline bool norm_rows_takes(const MoNorm& a, RowsCut& c) {
    const int cg = a.C / a.groups;
    c.one = a.S == 1 && cg > kWave;
    if (c.one ? cg > ROWS_MOST * kWave : (cg > kWave || a.S > ROWS_MOST * (kWave / cg))) return false;
    for (c.TT = 1; c.TT < kWave && c.TT < cg * a.S; c.TT *= 2) {}
    c.PL = c.one ? 1 : c.TT / cg;
    const int64_t each = c.one ? (cg + kWave - 1) / kWave : (a.S + c.PL - 1) / c.PL;
    c.R = each <= 1 ? 1 : each <= 4 ? 4 : ROWS_MOST;
    const int64_t fill = (int64_t)compute_units() * 8 * (NORM_THREADS / c.TT);   // teams
    c.rows = std::min<int64_t>(a.B, std::max<int64_t>(1, fill / a.groups));
    c.blocks = (int)((c.rows * a.groups * c.TT + NORM_THREADS - 1) / NORM_THREADS);
    return true;
}
inline int64_t norm_rows_work(const MoNorm& a, const RowsCut& c, bool backward) {   // in floats
    return backward && a.dweight ? (c.rows + NORM_SUM_ROWS) * 2 * a.C : 0;
}

template <class T, int R, bool ONE, int ACT> int norm_rows_run(const Rows& k, const RowsCut& c, bool backward, hipStream_t s) {
    if (backward) hipLaunchKernelGGL((k_norm_rows_back<T, R, ONE, ACT>), dim3(c.blocks), dim3(NORM_THREADS), 0, s, k);
    else hipLaunchKernelGGL((k_norm_rows<T, R, ONE, ACT>), dim3(c.blocks), dim3(NORM_THREADS), 0, s, k);
    return launched("k_norm_rows");
}
template <class T, int ACT> int norm_rows(const MoNorm& a, const RowsCut& c, bool backward, hipStream_t s) {
    const Rows k{a, a.C / a.groups, c.TT, c.PL, c.rows, backward && a.dweight ? (float*)a.work : nullptr};
    const int rc = c.one ? (c.R == 4 ? norm_rows_run<T, 4, true, ACT>(k, c, backward, s) : norm_rows_run<T, ROWS_MOST, true, ACT>(k, c, backward, s))
                 : c.R == 1 ? norm_rows_run<T, 1, false, ACT>(k, c, backward, s)
                 : c.R == 4 ? norm_rows_run<T, 4, false, ACT>(k, c, backward, s) : norm_rows_run<T, ROWS_MOST, false, ACT>(k, c, backward, s);
    return rc || !k.part ? rc : norm_colsum(a, k.part, c.rows, k.part + c.rows * 2 * a.C, s);
}

}  // namespace mo
