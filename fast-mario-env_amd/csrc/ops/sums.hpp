// Sums over lanes and over the rows that workgroups leave, in a fixed order.
#pragma once
#include "common.hpp"

namespace mo {

// x of the lane that DPP's control word names (within rows of 16).
template <int CTRL> __device__ __forceinline__ float dpp(float x) {
    return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), CTRL, 0xf, 0xf, true));
}
constexpr int DPP_XOR1 = 0xB1, DPP_XOR2 = 0x4E, DPP_MIRROR8 = 0x141, DPP_MIRROR16 = 0x140;   // (mirrored: l to 7 - l, l to 15 - l)

// Sums of M values over a wave's 64 lanes, each lane left with one of them: every step keeps half of the values in half of the lanes, so that
// 16 values cost 35 instructions and not 96 (47 with swaps alone). Within rows of 16 lanes a value's sum is written over the other's in the lanes that are its own
// (DPP's bank mask: two instructions a pair); rows are exchanged by permlane swaps (three). Lane l gets value sum_slot(l) of the M (4, 8,
// 12 or 16; a slot >= M holds nothing), lanes of equal slots the same sum.
__device__ __forceinline__ int sum_slot(int l, int M) {
    if (M <= 4) return ((l >> 3) & 1) | ((l >> 1) & 2);
    const int s = ((l >> 3) & 1) | ((l >> 1) & 2) | ((l >> 2) & 4);
    return M <= 8 ? s : s | ((l >> 2) & 8);
}
// x = x + (x of lane l ^ 8), y's likewise in the upper eight lanes of each row; then likewise four and four, the others mirrored. (An operand of DPP or a
// permlane swap may not have been written by the two instructions before: the nops at both ends, and the order between them. What is written before the
// last input is read shares no register with an input, equal or not: the `&`.)
__device__ __forceinline__ void row_sums4(float& x0, float x1, float& x2, float x3) {
    asm("s_nop 1\n\t"
        "v_add_f32_dpp %0, %0, %0 row_ror:8 row_mask:0xf bank_mask:0xf\n\tv_add_f32_dpp %1, %1, %1 row_ror:8 row_mask:0xf bank_mask:0xf\n\t"
        "v_add_f32_dpp %0, %2, %2 row_ror:8 row_mask:0xf bank_mask:0xc\n\tv_add_f32_dpp %1, %3, %3 row_ror:8 row_mask:0xf bank_mask:0xc\n\t"
        "s_nop 1\n\t"
        "v_add_f32_dpp %0, %0, %0 row_half_mirror row_mask:0xf bank_mask:0xf\n\t"
        "v_add_f32_dpp %0, %1, %1 row_half_mirror row_mask:0xf bank_mask:0xa\n\ts_nop 1"
        : "+&v"(x0), "+&v"(x2)
        : "v"(x1), "v"(x3));
}
__device__ __forceinline__ void row_sums8(float& x0, float x1, float& x2, float x3, float& x4, float x5, float& x6, float x7) {
    asm("s_nop 1\n\t"
        "v_add_f32_dpp %0, %0, %0 row_ror:8 row_mask:0xf bank_mask:0xf\n\tv_add_f32_dpp %1, %1, %1 row_ror:8 row_mask:0xf bank_mask:0xf\n\t"
        "v_add_f32_dpp %2, %2, %2 row_ror:8 row_mask:0xf bank_mask:0xf\n\tv_add_f32_dpp %3, %3, %3 row_ror:8 row_mask:0xf bank_mask:0xf\n\t"
        "v_add_f32_dpp %0, %4, %4 row_ror:8 row_mask:0xf bank_mask:0xc\n\tv_add_f32_dpp %1, %5, %5 row_ror:8 row_mask:0xf bank_mask:0xc\n\t"
        "v_add_f32_dpp %2, %6, %6 row_ror:8 row_mask:0xf bank_mask:0xc\n\tv_add_f32_dpp %3, %7, %7 row_ror:8 row_mask:0xf bank_mask:0xc\n\t"
        "v_add_f32_dpp %0, %0, %0 row_half_mirror row_mask:0xf bank_mask:0xf\n\tv_add_f32_dpp %2, %2, %2 row_half_mirror row_mask:0xf bank_mask:0xf\n\t"
        "v_add_f32_dpp %0, %1, %1 row_half_mirror row_mask:0xf bank_mask:0xa\n\tv_add_f32_dpp %2, %3, %3 row_half_mirror row_mask:0xf bank_mask:0xa\n\ts_nop 1"
        : "+&v"(x0), "+&v"(x2), "+&v"(x4), "+&v"(x6)
        : "v"(x1), "v"(x3), "v"(x5), "v"(x7));
}
template <int M> __device__ __forceinline__ float wave_sums(float (&v)[M]) {
    static_assert(M % 4 == 0 && M <= 16, "");
    typedef unsigned U2 __attribute__((ext_vector_type(2)));
    float r[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < M / 4; i += 2) {
        if (i + 1 < M / 4) {
            row_sums8(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3], v[4 * i + 4], v[4 * i + 5], v[4 * i + 6], v[4 * i + 7]);
            r[i + 1] = v[4 * i + 4];
        } else {
            row_sums4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
        }
        r[i] = v[4 * i];
    }
    if constexpr (M > 4) {                                    // rows 0 and 2 keep the first, rows 1 and 3 the second
        const auto rows = [](float a, float b) {
            const U2 x = __builtin_amdgcn_permlane16_swap(__float_as_uint(a), __float_as_uint(b), false, false);
            return __uint_as_float(x[0]) + __uint_as_float(x[1]);
        };
        r[0] = rows(r[0], r[1]);
        if constexpr (M > 8) r[2] = rows(r[2], r[3]);
    } else {
        const U2 x = __builtin_amdgcn_permlane16_swap(__float_as_uint(r[0]), __float_as_uint(r[0]), false, false);
        r[0] = __uint_as_float(x[0]) + __uint_as_float(x[1]);
    }
    const U2 x = __builtin_amdgcn_permlane32_swap(__float_as_uint(r[0]), __float_as_uint(M > 8 ? r[2] : r[0]), false, false);
    float sum = __uint_as_float(x[0]) + __uint_as_float(x[1]);
    sum += dpp<DPP_XOR2>(sum);
    return sum + dpp<DPP_XOR1>(sum);
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
