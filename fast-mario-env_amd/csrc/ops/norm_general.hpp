// Group norm with an activation, channels last: any channel and group counts, any sample size.
#pragma once
#include "common.hpp"

namespace mo {

// With h = (x - mean) rstd and z = weight h + bias:  y = act(z). Going back, dz = dy act'(z), dbias = sum dz, dweight = sum dz h
// and, with dh = weight dz,  dx = rstd (dh - mean(dh) - h mean(dh h)), the means over the group.
template <int ACT> __device__ __forceinline__ float act(float z) {
    if (ACT == MO_ACT_RELU) return z <= 0.f ? 0.f : z;   // (a NaN stays one)
    if (ACT == MO_ACT_SILU) return z * __builtin_amdgcn_rcpf(1.f + __expf(-z));
    return z;
}
template <int ACT> __device__ __forceinline__ float act_grad(float z) {
    if (ACT == MO_ACT_RELU) return z > 0.f ? 1.f : 0.f;
    if (ACT == MO_ACT_SILU) {
        const float s = __builtin_amdgcn_rcpf(1.f + __expf(-z));
        return s * (1.f + z * (1.f - s));
    }
    return 1.f;
}

// n values of mean `mean` and squared deviations `m2`, joined by another set (Chan et al.): no difference of large sums.
struct Moments {
    float n, mean, m2;
    __device__ __forceinline__ void join(const Moments& o) {
        if (o.n == 0.f) return;
        if (n == 0.f) { *this = o; return; }   // (the square of a large mean is infinite, and times no values a NaN)
        const float t = n + o.n;
        const float d = o.mean - mean, w = o.n / t;
        mean = fmaf(d, w, mean);
        m2 = m2 + o.m2 + d * d * n * w;
        n = t;
    }
};

// For samples that do not fit a team's registers. Three passes: the slabs' moments (back: sums), their joining, and the results, so x
// is read twice (back: x and dy), each time past the L2s (counters; the last-level cache may have it the second time). Measured, float32, 37 x
// 48 x 84 x 84 in 6 groups, in microseconds under the profiler: moments 17, their joining 4, results 21; back, sums 22, joining 5, results 28,
// the channels' sums 4; 97 in all without it.
// A sample is cut into slabs of `px` pixels; a block takes a slab. Its threads are LN lanes along the channels (V each) by
// pixel lanes, so a thread's channels stay its own.
struct NormCut {
    int64_t slabs, px;
    int nv, LN, PL;   // packs of V channels a pixel; channel lanes; pixel lanes
    bool by_group;    // a block sees whole pixels, and joins its channels' sums to the groups'
};

struct NormArgs {
    MoNorm a;
    NormCut c;
    float* part;      // per (sample, slab): [2][C], each channel's two sums
    float* group;     // per (sample, slab): [2][groups], each group's (by_group)
    float* means;     // (B, groups, 2): mean and rstd; going back, mean(dh) and mean(dh h)
};

constexpr int NORM_THREADS = 256;

// Each channel's (or group's) mean and squared deviations over a slab. A thread sums runs of NORM_RUN values about their first, and
// the runs' and the threads' sets are joined as moments. A run's sum of squares about one of its n values is at most n times that
// about its mean, so a far value costs a run n roundings at most, and a large mean none. (About a thread's first value of all, one that
// is far off took a thousandth of the variance along.)
constexpr int NORM_RUN = 16;
template <class T, int V>
__global__ void __launch_bounds__(NORM_THREADS) k_norm_moments(NormArgs k) {
    __shared__ float sm[NORM_THREADS][V], s2[NORM_THREADS][V], sn[NORM_THREADS];
    const MoNorm& a = k.a;
    const int64_t at_block = block_here(), b = at_block / k.c.slabs, slab = at_block % k.c.slabs, p0 = slab * k.c.px, p1 = min(p0 + k.c.px, a.S);
    if (b >= a.B) return;
    const int t = threadIdx.x, pl = t / k.c.LN;
    float* part = k.part + at_block * 2 * a.C;
    for (int c0 = 0; c0 < k.c.nv; c0 += k.c.LN) {
        const int cv = c0 + t % k.c.LN;
        const bool live = pl < k.c.PL && cv < k.c.nv;
        float mean[V] = {}, m2[V] = {}, n = 0.f;
        if (live)
            for (int64_t p = p0 + pl; p < p1;) {
                float about[V], sum[V] = {}, sq[V] = {}, run = 0.f;
#pragma unroll 4
                for (int j = 0; j < NORM_RUN && p < p1; j++, p += k.c.PL, run += 1.f) {
                    const Pack<T, V> x = *(const Pack<T, V>*)((const T*)a.x + (b * a.S + p) * a.C + cv * V);
#pragma unroll
                    for (int i = 0; i < V; i++) {
                        if (j == 0) about[i] = as_f32(x.v[i]);
                        const float d = as_f32(x.v[i]) - about[i];
                        sum[i] += d;
                        sq[i] = fmaf(d, d, sq[i]);
                    }
                }
                n += run;
                const float r = 1.f / run, w = run / n, both = (n - run) * w;
#pragma unroll
                for (int i = 0; i < V; i++) {
                    const float e = sum[i] * r, here = about[i] + e;
                    const float d = n == run ? 0.f : here - mean[i];
                    mean[i] = n == run ? here : fmaf(d, w, mean[i]);
                    m2[i] += fmaxf(fmaf(-e, sum[i], sq[i]), 0.f) + (sq[i] - sq[i]) + d * d * both;   // (what is not finite stays so)
                }
            }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < V; i++) { sm[t][i] = mean[i]; s2[t][i] = m2[i]; }
        sn[t] = n;
        for (int m = 1; m < k.c.PL; m *= 2) {                  // pixel lanes j and j + m
            __syncthreads();
            if (live && pl % (2 * m) == 0 && pl + m < k.c.PL) {
                const int o = t + m * k.c.LN;
                const float na = sn[t], nb = sn[o], nt = na + nb, w = nt > 0.f ? nb / nt : 0.f;
#pragma unroll
                for (int i = 0; i < V; i++) {
                    const float d = sm[o][i] - sm[t][i];
                    if (nb > 0.f) {
                        sm[t][i] = fmaf(d, w, sm[t][i]);
                        s2[t][i] += s2[o][i] + d * d * na * w;
                    }
                }
                sn[t] = nt;
            }
        }
        if (!k.c.by_group) {
            if (live && pl == 0)
#pragma unroll
                for (int i = 0; i < V; i++) {
                    part[cv * V + i] = sm[t][i];
                    part[a.C + cv * V + i] = s2[t][i];
                }
            continue;
        }
        __syncthreads();
        const int cg = a.C / a.groups;                         // channels of one count: a mean of means, about the first
        float* group = k.group + at_block * 2 * a.groups;
        for (int g = t / kWave; g < a.groups; g += NORM_THREADS / kWave) {
            const float m0 = sm[g * cg / V][g * cg % V];
            float mean = 0.f, m2 = 0.f;
            for (int c = g * cg + t % kWave; c < (g + 1) * cg; c += kWave) mean += sm[c / V][c % V] - m0;
            for (int s = 1; s < kWave; s *= 2) mean += __shfl_xor(mean, s);
            mean = m0 + mean / (float)cg;
            for (int c = g * cg + t % kWave; c < (g + 1) * cg; c += kWave) {
                const float d = sm[c / V][c % V] - mean;
                m2 += s2[c / V][c % V] + sn[0] * d * d;
            }
            for (int s = 1; s < kWave; s *= 2) m2 += __shfl_xor(m2, s);
            if (t % kWave == 0) {
                group[g] = mean;
                group[a.groups + g] = m2;
            }
        }
    }
}

// Mean and rstd of a sample's group, a block each, from the moments of every slab (of its channels, or its own).
__global__ void __launch_bounds__(NORM_THREADS) k_norm_means(NormArgs k) {
    __shared__ Moments of[NORM_THREADS];
    const MoNorm& a = k.a;
    const int64_t bg = block_here(), b = bg / a.groups;
    if (b >= a.B) return;
    const int g = (int)(bg % a.groups), cg = a.C / a.groups, t = threadIdx.x;
    const int per = k.c.by_group ? 1 : cg, width = k.c.by_group ? a.groups : a.C;
    const float* from = (k.c.by_group ? k.group : k.part) + b * k.c.slabs * 2 * width + g * per;
    Moments m{0.f, 0.f, 0.f};
    for (int64_t i = t; i < k.c.slabs * per; i += NORM_THREADS) {
        const int64_t slab = i / per;
        const float* p = from + slab * 2 * width + i % per;
        m.join({(float)(min((slab + 1) * k.c.px, a.S) - slab * k.c.px) * (float)(cg / per), p[0], p[width]});
    }
    of[t] = m;
    for (int s = 1; s < NORM_THREADS; s *= 2) {
        __syncthreads();
        if (t % (2 * s) == 0) of[t].join(of[t + s]);
    }
    if (t == 0) {
        k.means[2 * bg] = of[0].mean;
        k.means[2 * bg + 1] = 1.f / sqrtf(of[0].m2 / of[0].n + a.eps);
    }
}

template <class T, int V, int ACT>
__global__ void __launch_bounds__(NORM_THREADS) k_norm_apply(NormArgs k) {
    const MoNorm& a = k.a;
    const int64_t at_block = block_here(), b = at_block / k.c.slabs, slab = at_block % k.c.slabs, p0 = slab * k.c.px, p1 = min(p0 + k.c.px, a.S);
    if (b >= a.B) return;
    const int t = threadIdx.x, pl = t / k.c.LN, cg = a.C / a.groups;
    if (pl >= k.c.PL) return;
    for (int cv = t % k.c.LN; cv < k.c.nv; cv += k.c.LN) {
        float w[V], s[V], mean[V];                        // z = (x - mean) w + s
#pragma unroll
        for (int i = 0; i < V; i++) {
            const int c = cv * V + i;
            const float* m = k.means + 2 * (b * a.groups + c / cg);
            mean[i] = m[0];
            w[i] = m[1] * (a.weight ? a.weight[c] : 1.f);
            s[i] = a.bias ? a.bias[c] : 0.f;
        }
        for (int64_t p = p0 + pl; p < p1; p += k.c.PL) {
            const int64_t at = (b * a.S + p) * a.C + cv * V;
            Pack<T, V> x = *(const Pack<T, V>*)((const T*)a.x + at);
#pragma unroll
            for (int i = 0; i < V; i++) x.v[i] = as<T>(act<ACT>(fmaf(as_f32(x.v[i]) - mean[i], w[i], s[i])));
            stream((Pack<T, V>*)((T*)a.y + at), x);
        }
    }
}

// Each channel's sums of dz h and of dz over a slab, into part, and each group's of dh and dh h.
template <class T, int V, int ACT>
__global__ void __launch_bounds__(NORM_THREADS) k_norm_sums(NormArgs k) {
    __shared__ float sw[NORM_THREADS][V], sb[NORM_THREADS][V];
    const MoNorm& a = k.a;
    const int64_t at_block = block_here(), b = at_block / k.c.slabs, slab = at_block % k.c.slabs, p0 = slab * k.c.px, p1 = min(p0 + k.c.px, a.S);
    if (b >= a.B) return;
    const int t = threadIdx.x, pl = t / k.c.LN, cg = a.C / a.groups;
    float* part = k.part + at_block * 2 * a.C;
    for (int c0 = 0; c0 < k.c.nv; c0 += k.c.LN) {
        const int cv = c0 + t % k.c.LN;
        const bool live = pl < k.c.PL && cv < k.c.nv;
        float dw[V] = {}, db[V] = {};
        if (live) {
            float w[V], s[V], mean[V], r[V];
#pragma unroll
            for (int i = 0; i < V; i++) {
                const int c = cv * V + i;
                const float* m = a.stats + 2 * (b * a.groups + c / cg);
                mean[i] = m[0];
                r[i] = m[1];
                w[i] = a.weight ? a.weight[c] : 1.f;
                s[i] = a.bias ? a.bias[c] : 0.f;
            }
            for (int64_t p = p0 + pl; p < p1; p += k.c.PL) {
                const int64_t at = (b * a.S + p) * a.C + cv * V;
                const Pack<T, V> x = *(const Pack<T, V>*)((const T*)a.x + at), dy = *(const Pack<T, V>*)((const T*)a.dy + at);
#pragma unroll
                for (int i = 0; i < V; i++) {
                    const float h = (as_f32(x.v[i]) - mean[i]) * r[i], dz = as_f32(dy.v[i]) * act_grad<ACT>(fmaf(h, w[i], s[i]));
                    dw[i] = fmaf(dz, h, dw[i]);
                    db[i] += dz;
                }
            }
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < V; i++) { sw[t][i] = dw[i]; sb[t][i] = db[i]; }
        for (int m = 1; m < k.c.PL; m *= 2) {                  // pixel lanes j and j + m
            __syncthreads();
            if (live && pl % (2 * m) == 0 && pl + m < k.c.PL)
#pragma unroll
                for (int i = 0; i < V; i++) {
                    sw[t][i] += sw[t + m * k.c.LN][i];
                    sb[t][i] += sb[t + m * k.c.LN][i];
                }
        }
        if (live && pl == 0 && (a.dweight || !k.c.by_group))
#pragma unroll
            for (int i = 0; i < V; i++) {
                part[cv * V + i] = sw[t][i];
                part[a.C + cv * V + i] = sb[t][i];
            }
        if (!k.c.by_group) continue;
        __syncthreads();
        float* group = k.group + at_block * 2 * a.groups;
        for (int g = t / kWave; g < a.groups; g += NORM_THREADS / kWave) {
            float m1 = 0.f, m2 = 0.f;
            for (int c = g * cg + t % kWave; c < (g + 1) * cg; c += kWave) {
                const float w = a.weight ? a.weight[c] : 1.f;
                m1 = fmaf(w, sb[c / V][c % V], m1);
                m2 = fmaf(w, sw[c / V][c % V], m2);
            }
            for (int s = 1; s < kWave; s *= 2) { m1 += __shfl_xor(m1, s); m2 += __shfl_xor(m2, s); }
            if (t % kWave == 0) {
                group[g] = m1;
                group[a.groups + g] = m2;
            }
        }
    }
}

// mean(dh) and mean(dh h) of a sample's group, a block each, from the sums of every slab (of its channels, or its own).
__global__ void __launch_bounds__(NORM_THREADS) k_norm_dmeans(NormArgs k) {
    __shared__ float s1[NORM_THREADS], s2[NORM_THREADS];
    const MoNorm& a = k.a;
    const int64_t bg = block_here(), b = bg / a.groups;
    if (b >= a.B) return;
    const int g = (int)(bg % a.groups), cg = a.C / a.groups, t = threadIdx.x;
    float m1 = 0.f, m2 = 0.f;
    if (k.c.by_group)
        for (int64_t slab = t; slab < k.c.slabs; slab += NORM_THREADS) {
            const float* p = k.group + (b * k.c.slabs + slab) * 2 * a.groups + g;
            m1 += p[0];
            m2 += p[a.groups];
        }
    else
        for (int64_t i = t; i < k.c.slabs * cg; i += NORM_THREADS) {
            const int c = g * cg + (int)(i % cg);
            const float* p = k.part + (b * k.c.slabs + i / cg) * 2 * a.C + c;
            const float w = a.weight ? a.weight[c] : 1.f;
            m2 = fmaf(w, p[0], m2);
            m1 = fmaf(w, p[a.C], m1);
        }
    s1[t] = m1;
    s2[t] = m2;
    for (int s = NORM_THREADS / 2; s; s /= 2) {
        __syncthreads();
        if (t < s) { s1[t] += s1[t + s]; s2[t] += s2[t + s]; }
    }
    if (t == 0) {
        const float by = 1.f / ((float)a.S * (float)cg);
        k.means[2 * bg] = s1[0] * by;
        k.means[2 * bg + 1] = s2[0] * by;
    }
}

template <class T, int V, int ACT>
__global__ void __launch_bounds__(NORM_THREADS) k_norm_dx(NormArgs k) {
    const MoNorm& a = k.a;
    const int64_t at_block = block_here(), b = at_block / k.c.slabs, slab = at_block % k.c.slabs, p0 = slab * k.c.px, p1 = min(p0 + k.c.px, a.S);
    if (b >= a.B) return;
    const int t = threadIdx.x, pl = t / k.c.LN, cg = a.C / a.groups;
    if (pl >= k.c.PL) return;
    for (int cv = t % k.c.LN; cv < k.c.nv; cv += k.c.LN) {
        float w[V], s[V], mean[V], r[V], m1[V], m2[V];
#pragma unroll
        for (int i = 0; i < V; i++) {
            const int c = cv * V + i;
            const int64_t g = 2 * (b * a.groups + c / cg);
            mean[i] = a.stats[g];
            r[i] = a.stats[g + 1];
            m1[i] = k.means[g];
            m2[i] = k.means[g + 1];
            w[i] = a.weight ? a.weight[c] : 1.f;
            s[i] = a.bias ? a.bias[c] : 0.f;
        }
        for (int64_t p = p0 + pl; p < p1; p += k.c.PL) {
            const int64_t at = (b * a.S + p) * a.C + cv * V;
            const Pack<T, V> x = *(const Pack<T, V>*)((const T*)a.x + at);
            Pack<T, V> dy = *(const Pack<T, V>*)((const T*)a.dy + at);
#pragma unroll
            for (int i = 0; i < V; i++) {
                const float h = (as_f32(x.v[i]) - mean[i]) * r[i], dz = as_f32(dy.v[i]) * act_grad<ACT>(fmaf(h, w[i], s[i]));
                dy.v[i] = as<T>(r[i] * (w[i] * dz - m1[i] - h * m2[i]));
            }
            stream((Pack<T, V>*)((T*)a.dx + at), dy);
        }
    }
}

// Sums the rows of `in` (rows, cols) that belong to block row blockIdx.y: 16 columns by 64 row lanes, each eight loads ahead,
// joined in order. The last round (one block row) writes the first half of the columns to dweight and the rest to dbias.
constexpr int SUM_COLS = 16, SUM_LANES = 64;
__global__ void __launch_bounds__(SUM_COLS * SUM_LANES) k_norm_colsum(const float* in, int64_t rows, int cols, float* out, float* dweight,
                                                                     float* dbias) {
    __shared__ float s[SUM_LANES][SUM_COLS];
    const int cl = threadIdx.x % SUM_COLS, c = blockIdx.x * SUM_COLS + cl, rl = threadIdx.x / SUM_COLS;
    const int64_t step = (int64_t)SUM_LANES * gridDim.y;
    float sum = 0.f;
    if (c < cols)
        for (int64_t r = (int64_t)blockIdx.y * SUM_LANES + rl; r < rows; r += 8 * step) {
            float x[8];
#pragma unroll
            for (int i = 0; i < 8; i++) x[i] = r + i * step < rows ? in[(r + i * step) * cols + c] : 0.f;
#pragma unroll
            for (int i = 0; i < 8; i++) sum += x[i];
        }
    s[rl][cl] = sum;
    for (int m = SUM_LANES / 2; m; m /= 2) {
        __syncthreads();
        if (rl < m) s[rl][cl] += s[rl + m][cl];
    }
    if (rl || c >= cols) return;
    sum = s[0][cl];
    if (out) out[(int64_t)blockIdx.y * cols + c] = sum;
    else if (c < cols / 2) dweight[c] = sum;
    else dbias[c - cols / 2] = sum;
}

constexpr int NORM_SUM_ROWS = 64;   // rows that the first round of column sums leaves

// rows of (2, C) sums -> dweight, dbias, in two rounds where a block would go through many rows (200,000 of 60 columns: 310 us less
// of a gradient than in one; 1,024 rows of 1,024 columns: 8 us more); `spare` holds NORM_SUM_ROWS rows.
inline int norm_colsum(const MoNorm& a, const float* rows_of, int64_t rows, float* spare, hipStream_t s) {
    const int cols = 2 * a.C;
    const unsigned blocks = (unsigned)((cols + SUM_COLS - 1) / SUM_COLS);
    if (rows > 4096) {
        hipLaunchKernelGGL(k_norm_colsum, dim3(blocks, NORM_SUM_ROWS), dim3(SUM_COLS * SUM_LANES), 0, s, rows_of, rows, cols, spare, nullptr, nullptr);
        if (launched("k_norm_colsum")) return -1;
        rows_of = spare;
        rows = NORM_SUM_ROWS;
    }
    hipLaunchKernelGGL(k_norm_colsum, dim3(blocks), dim3(SUM_COLS * SUM_LANES), 0, s, rows_of, rows, cols, nullptr, a.dweight, a.dbias);
    return launched("k_norm_colsum");
}

// ---- host side
inline bool norm_wide(const MoNorm& a) {   // 8 channels an access (of 16 bytes, or two of them)
    uintptr_t p = (uintptr_t)a.x | (uintptr_t)a.y | (uintptr_t)a.dy | (uintptr_t)a.dx;
    return a.C % 8 == 0 && p % 16 == 0;
}

// Slabs: enough blocks for the chip where samples are few, and at least 16 KB of a sample in each. (37 x 48 x 84 x 84 float32, forward and
// gradient: 97 us with up to 1,024 blocks, 105 with 2,048, 119 with 4,096; 500 x 32 x 84 x 84 bf16 366, 366 and 374.)
inline NormCut norm_cut(const MoNorm& a, int V) {
    NormCut c;
    const int64_t per_px = (int64_t)a.C * (a.dtype == MO_BF16 ? 2 : 4);
    const int64_t most = std::max<int64_t>(1, a.S * per_px / (16 << 10)), want = std::max<int64_t>(1, 1024 / std::max<int64_t>(1, a.B));
    c.px = (a.S + std::min(most, want) - 1) / std::min(most, want);
    c.slabs = (a.S + c.px - 1) / c.px;
    c.nv = a.C / V;
    c.LN = std::min(c.nv, NORM_THREADS);
    c.PL = NORM_THREADS / c.LN;
    c.by_group = c.nv == c.LN;
    return c;
}

struct NormWork { int64_t part, group, means, spare, total; };   // in floats
inline NormWork norm_general_work(const MoNorm& a, const NormCut& c, bool backward) {
    NormWork w;
    w.part = c.by_group && !(backward && a.dweight) ? 0 : a.B * c.slabs * 2 * a.C;
    w.group = c.by_group ? a.B * c.slabs * 2 * a.groups : 0;
    w.means = a.B * a.groups * 2;
    w.spare = backward ? (int64_t)NORM_SUM_ROWS * 2 * a.C : 0;
    w.total = w.part + w.group + w.means + w.spare;
    return w;
}

template <class T, int V, int ACT> int norm_general(const MoNorm& a, bool backward, hipStream_t s) {
    NormArgs k{a, norm_cut(a, V), nullptr, nullptr, nullptr};
    const NormWork w = norm_general_work(a, k.c, backward);
    k.part = (float*)a.work;
    k.group = k.part + w.part;
    k.means = k.group + w.group;
    const dim3 grid = grid_of(a.B * k.c.slabs), per_group = grid_of(a.B * a.groups);
    if (!backward) {
        if (a.stats) k.means = a.stats;
        hipLaunchKernelGGL((k_norm_moments<T, V>), grid, dim3(NORM_THREADS), 0, s, k);
        hipLaunchKernelGGL(k_norm_means, per_group, dim3(NORM_THREADS), 0, s, k);
        hipLaunchKernelGGL((k_norm_apply<T, V, ACT>), grid, dim3(NORM_THREADS), 0, s, k);
        return launched("k_norm_apply");
    }
    hipLaunchKernelGGL((k_norm_sums<T, V, ACT>), grid, dim3(NORM_THREADS), 0, s, k);
    hipLaunchKernelGGL(k_norm_dmeans, per_group, dim3(NORM_THREADS), 0, s, k);
    hipLaunchKernelGGL((k_norm_dx<T, V, ACT>), grid, dim3(NORM_THREADS), 0, s, k);
    if (launched("k_norm_dx")) return -1;
    return a.dweight ? norm_colsum(a, k.part, a.B * k.c.slabs, k.means + w.means, s) : 0;
}

}  // namespace mo
