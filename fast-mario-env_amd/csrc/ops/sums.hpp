// Sums over lanes and over the rows that workgroups leave, in a fixed order.
#pragma once
#include "common.hpp"

namespace mo {

// x of the lane that DPP's control word names (within rows of 16).
template <int CTRL> __device__ __forceinline__ float dpp(float x) {
    return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), CTRL, 0xf, 0xf, true));
}
constexpr int DPP_XOR1 = 0xB1, DPP_XOR2 = 0x4E, DPP_MIRROR8 = 0x141, DPP_XOR8 = 0x128;   // (mirrored in eights: l to 7 - l)

// Sums of M values over a wave's 64 lanes, each lane left with one of them: every step sends half of the values to the other half of the
// lanes, so that M values cost about 3 M instructions and not 12 M. Lane l gets value sum_slot(l) of the M (4, 8, 12 or 16; a slot >= M
// holds nothing), lanes of equal slots the same sum.
__device__ __forceinline__ int sum_slot(int l, int M) {
    const int s = ((l >> 5) & 1) | ((l >> 3) & 2) | ((l >> 1) & 4) | ((l << 1) & 8);
    return M <= 4 ? s & 3 : M <= 8 ? s & 7 : s;
}
template <int M> __device__ __forceinline__ float wave_sums(float (&v)[M]) {
    static_assert(M % 4 == 0 && M <= 16, "");
    const int l = threadIdx.x % kWave;
    float a[M / 2], b[M / 4];
    typedef unsigned U2 __attribute__((ext_vector_type(2)));
#pragma unroll
    for (int i = 0; i < M / 2; i++) {
        const U2 x = __builtin_amdgcn_permlane32_swap(__float_as_uint(v[2 * i]), __float_as_uint(v[2 * i + 1]), false, false);
        a[i] = __uint_as_float(x[0]) + __uint_as_float(x[1]);
    }
#pragma unroll
    for (int i = 0; i < M / 4; i++) {
        const U2 x = __builtin_amdgcn_permlane16_swap(__float_as_uint(a[2 * i]), __float_as_uint(a[2 * i + 1]), false, false);
        b[i] = __uint_as_float(x[0]) + __uint_as_float(x[1]);
    }
    float r;
    if constexpr (M == 4) {
        r = b[0] + dpp<DPP_XOR8>(b[0]);
        r += dpp<DPP_MIRROR8>(r);
    } else {
        const float b3 = M == 16 ? b[M / 4 - 1] : 0.f;
        const float c0 = (l & 8 ? b[1] : b[0]) + dpp<DPP_XOR8>(l & 8 ? b[0] : b[1]);
        if constexpr (M == 8) {
            r = c0 + dpp<DPP_MIRROR8>(c0);
        } else {
            const float c1 = (l & 8 ? b3 : b[2]) + dpp<DPP_XOR8>(l & 8 ? b[2] : b3);
            r = (l & 4 ? c1 : c0) + dpp<DPP_MIRROR8>(l & 4 ? c0 : c1);
        }
    }
    r += dpp<DPP_XOR2>(r);
    return r + dpp<DPP_XOR1>(r);
}

// Column sums of parameters' gradients: `rows` rows of `lines` x C floats, whose first `S` lines are the columns of `first` (C, S) and the
// lines from `tail` on `second` (C) and `third` (C); each may be null. A block takes 64 columns and 1 / gridDim.y of the rows; where that is
// not all of them, its sums are a row of `part`, and a second launch takes those.
struct ColumnSums {
    const float* from;
    float* part;
    int64_t rows;
    int lines, C, S, tail;
    float *first, *second, *third;
};
constexpr int SUM_THREADS = 1024, SUM_LANES = SUM_THREADS / kWave;

__global__ void __launch_bounds__(SUM_THREADS) k_column_sums(ColumnSums a) {
    __shared__ float s[SUM_LANES][kWave];
    const int lane = threadIdx.x % kWave, r0 = threadIdx.x / kWave;
    const int64_t M = (int64_t)a.lines * a.C, col = (int64_t)blockIdx.x * kWave + lane;
    const int64_t each = (a.rows + gridDim.y - 1) / gridDim.y, end = min(a.rows, (blockIdx.y + 1) * each);
    float x[4] = {0.f, 0.f, 0.f, 0.f};
    if (col < M) {
        int64_t r = blockIdx.y * each + r0;
        for (; r + 3 * SUM_LANES < end; r += 4 * SUM_LANES)
#pragma unroll
            for (int i = 0; i < 4; i++) x[i] += a.from[(r + i * SUM_LANES) * M + col];
        for (; r < end; r += SUM_LANES) x[0] += a.from[r * M + col];
    }
    s[r0][lane] = (x[0] + x[1]) + (x[2] + x[3]);
    for (int m = SUM_LANES / 2; m; m /= 2) {
        __syncthreads();
        if (r0 < m) s[r0][lane] += s[r0 + m][lane];
    }
    if (r0 || col >= M) return;
    const float sum = s[0][lane];
    if (gridDim.y > 1) {
        a.part[blockIdx.y * M + col] = sum;
        return;
    }
    const int line = (int)(col / a.C), c = (int)(col % a.C);
    if (line < a.S) {
        if (a.first) a.first[(int64_t)c * a.S + line] = sum;
    } else if (line >= a.tail) {
        float* to = line == a.tail ? a.second : a.third;
        if (to) to[c] = sum;
    }
}
constexpr int SUM_PARTS = 16;
inline int64_t column_parts(int64_t rows) { return rows >= 16 * SUM_PARTS ? SUM_PARTS : 1; }   // (fewer rows: one launch is enough)
inline int64_t column_sums_work(int64_t rows, int lines, int C) { return column_parts(rows) > 1 ? SUM_PARTS * (int64_t)lines * C : 0; }
inline int column_sums(ColumnSums a, hipStream_t s) {
    const unsigned blocks = (unsigned)(((int64_t)a.lines * a.C + kWave - 1) / kWave), parts = (unsigned)column_parts(a.rows);
    hipLaunchKernelGGL(k_column_sums, dim3(blocks, parts), dim3(SUM_THREADS), 0, s, a);
    if (parts > 1) {
        a.from = a.part;
        a.rows = parts;
        hipLaunchKernelGGL(k_column_sums, dim3(blocks), dim3(SUM_THREADS), 0, s, a);
    }
    return launched("k_column_sums");
}

}  // namespace mo
