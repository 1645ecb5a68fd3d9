// 16 x 16 matrix-instruction tiles whose operands lie in LDS, for bf16 (one 16x16x32 product) and float32 (eight 16x16x4).
#pragma once
#include "common.hpp"

namespace mo {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef short i16x4 __attribute__((ext_vector_type(4)));

// An operand of a product over 32 indices: lane l has row (of A) or column (of B) l % 16 and the indices 8 (l / 16) + 0..7.
template <class T> struct Frag;
template <> struct Frag<bf16> { bf16x8 v; };
template <> struct Frag<float> { float v[8]; };

// acc (16 x 16; lane l has column l % 16 and rows 4 (l / 16) + 0..3) += A B
__device__ __forceinline__ void mma(f32x4& acc, const Frag<bf16>& a, const Frag<bf16>& b) {
    acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a.v, b.v, acc, 0, 0, 0);
}
__device__ __forceinline__ void mma(f32x4& acc, const Frag<float>& a, const Frag<float>& b) {
#pragma unroll
    for (int i = 0; i < 8; i++) acc = __builtin_amdgcn_mfma_f32_16x16x4f32(a.v[i], b.v[i], acc, 0, 0, 0);
}

// A tile in LDS of W elements a row, in 16-byte pieces. The pieces of a row are exchanged among each other by the row's number,
// so that the same piece of eight neighbouring rows, and two neighbouring pieces of four, lie in different banks: the pieces come
// straight from memory to where they are read, and rows need no padding.
template <class T, int W> struct Tile {
    static constexpr int EPV = 16 / sizeof(T), PIECES = W / EPV;
    static_assert(PIECES >= 4, "");
    T* p;
    static __device__ __forceinline__ unsigned turn(unsigned row) {
        return PIECES == 4 ? (row & 2) | ((row >> 2) & 1) : ((row & 3) << 1) | ((row >> 2) & 1);
    }
    __device__ __forceinline__ T* at(unsigned row, unsigned col) const {
        return p + (row * W + (((col / EPV) ^ turn(row)) * EPV | (col % EPV)));
    }

    // indices along the rows: `row` the operand's first, its indices from col
    __device__ __forceinline__ Frag<T> along(unsigned row, unsigned col, unsigned lane) const;
    // indices down the rows from `row`; the operand's rows or columns are the tile's columns from col, or (SPREAD) four of each
    // eight: column c of the operand is col + 8 (c / 4) + c % 4
    template <bool SPREAD = false> __device__ __forceinline__ Frag<T> down(unsigned row, unsigned col, unsigned lane) const;
};
template <class T, int W> __device__ __forceinline__ Frag<T> Tile<T, W>::along(unsigned row, unsigned col, unsigned lane) const {
    const unsigned r = row + lane % 16, c = col + 8 * (lane / 16);
    if constexpr (sizeof(T) == 2) {
        return {*(const bf16x8*)at(r, c)};
    } else {
        Frag<T> f;
        *(f32x4*)f.v = *(const f32x4*)at(r, c);
        *(f32x4*)(f.v + 4) = *(const f32x4*)at(r, c + 4);
        return f;
    }
}
template <class T, int W> template <bool SPREAD> __device__ __forceinline__ Frag<T> Tile<T, W>::down(unsigned row, unsigned col, unsigned lane) const {
    const unsigned g = lane / 16, i = lane % 16;
    if constexpr (sizeof(T) == 2) {   // the transposing LDS read: 16 lanes read four neighbours of each of 4 rows and get a column each
        typedef __attribute__((address_space(3))) i16x4* Lds;
        const unsigned r = row + 8 * g + i / 4, c = col + (i % 4) * (SPREAD ? 8 : 4);
        union { i16x4 h[2]; Frag<bf16> f; } u;
        u.h[0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((Lds)at(r, c));
        u.h[1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((Lds)at(r + 4, c));
        return u.f;
    } else {
        const unsigned c = col + (SPREAD ? 8 * (i / 4) + i % 4 : i);
        Frag<T> f;
#pragma unroll
        for (int e = 0; e < 8; e++) f.v[e] = *at(row + 8 * g + e, c);
        return f;
    }
}

// Accumulator tiles as an operand in place. A matrix's rows are dealt to its tiles so that this needs no exchange between lanes:
// row 4 g + r of tile t is row acc_row(t, g, r), and tiles 2 b and 2 b + 1 of a lane are its eight indices of block b. (An
// operand that makes such a tile takes its columns SPREAD.)
__device__ __forceinline__ constexpr int acc_row(int t, int g, int r) { return 32 * (t / 2) + 8 * g + 4 * (t % 2) + r; }
__device__ __forceinline__ constexpr int acc_col(int t) { return 32 * (t / 2) + 4 * (t % 2); }   // its first column there
__device__ __forceinline__ Pack<float, 4> pack4(const f32x4& x, float) { return *(const Pack<float, 4>*)&x; }
__device__ __forceinline__ Pack<bf16, 4> pack4(const f32x4& x, bf16) {   // two conversions an instruction
    const bf16x4 y = __builtin_convertvector(x, bf16x4);
    return *(const Pack<bf16, 4>*)&y;
}

// What a product takes from another product or from a state goes in as two bf16 parts, 16 bits of significand: with one, each of
// the sums that go into a result added a rounding of 2^-9 to the result's own (0.0024 of a result's norm in all, 0.0017 for the
// rounding of the result alone). The second part of what has overflowed or is not finite is 0, so that an infinity stays one.
// float32 is a part of its own.
template <class T> constexpr int kHalves = 1;
template <> inline constexpr int kHalves<bf16> = 2;

__device__ __forceinline__ void halves4(const f32x4& x, Pack<float, 4> (&part)[1]) { part[0] = pack4(x, 0.f); }
__device__ __forceinline__ void halves4(const f32x4& x, Pack<bf16, 4> (&part)[2]) {
    part[0] = pack4(x, bf16{});
    f32x4 rest;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        rest[i] = x[i] - (float)part[0].v[i];
        rest[i] = fabsf(rest[i]) < INFINITY ? rest[i] : 0.f;
    }
    part[1] = pack4(rest, bf16{});
}
template <class T> __device__ __forceinline__ void halves(const f32x4& a, const f32x4& b, Frag<T> (&part)[kHalves<T>]) {
    Pack<T, 4> x[kHalves<T>], y[kHalves<T>];
    halves4(a, x);
    halves4(b, y);
#pragma unroll
    for (int p = 0; p < kHalves<T>; p++) {
        union { Pack<T, 4> h[2]; Frag<T> f; } u{};
        u.h[0] = x[p];
        u.h[1] = y[p];
        part[p] = u.f;
    }
}

// The scores of a chunk's L steps with each other, on and below the diagonal, in LDS: tiles of 32 x 32 from the first row of blocks on.
template <class T, int L> struct Scores {
    static constexpr int SIZE = L * (L + 32) / 2;
    Tile<T, 32> t;
    static __device__ __forceinline__ unsigned row(unsigned i, unsigned j) {
        return L == 32 ? i : (i < 32 ? i : j < 32 ? i : i + 32);
    }
    __device__ __forceinline__ T* at(unsigned i, unsigned j) const { return t.at(row(i, j), j % 32); }
    __device__ __forceinline__ Frag<T> along(unsigned i, unsigned j, unsigned lane) const { return t.along(row(i, j), 0, lane); }
    __device__ __forceinline__ Frag<T> down(unsigned i, unsigned j, unsigned lane) const { return t.down(row(i, j), j % 32, lane); }
};
template <class T, int L> struct ScoreParts {
    Scores<T, L> part[kHalves<T>];
    __device__ __forceinline__ explicit ScoreParts(T* p) {
#pragma unroll
        for (int i = 0; i < kHalves<T>; i++) part[i].t.p = p + i * Scores<T, L>::SIZE;
    }
    __device__ __forceinline__ void put(unsigned i, unsigned j, const f32x4& x) const {   // four neighbours of a row
        Pack<T, 4> y[kHalves<T>];
        halves4(x, y);
#pragma unroll
        for (int p = 0; p < kHalves<T>; p++) *(Pack<T, 4>*)part[p].at(i, j) = y[p];
    }
    __device__ __forceinline__ float get(unsigned i, unsigned j) const {
        float x = as_f32(*part[0].at(i, j));
        if (kHalves<T> == 2) x += as_f32(*part[kHalves<T> - 1].at(i, j));
        return x;
    }
};

// The parts of w B, w a factor for each index, that keep float32's precision in products with bf16 operands: bf16 parts of 8 bits
// of significand each, three of which leave at most 2^-26 of it.
__device__ __forceinline__ void scaled_parts(const Frag<bf16>& b, const float* w, Frag<bf16>* part) {
    union { uint4 u; Frag<bf16> f; } in{};
    in.f = b;
    const uint32_t word[4] = {in.u.x, in.u.y, in.u.z, in.u.w};
#pragma unroll
    for (int h = 0; h < 2; h++) {
        f32x4 x;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const uint32_t y = word[2 * h + i / 2];
            x[i] = w[4 * h + i] * __uint_as_float(i % 2 ? y & 0xffff0000u : y << 16);
        }
#pragma unroll
        for (int p = 0; p < 3; p++) {
            union { bf16x4 v; uint2 u; } y{};
            y.v = __builtin_convertvector(x, bf16x4);
            ((uint2*)&part[p])[h] = y.u;
            if (p < 2) {
                x[0] -= __uint_as_float(y.u.x << 16);
                x[1] -= __uint_as_float(y.u.x & 0xffff0000u);
                x[2] -= __uint_as_float(y.u.y << 16);
                x[3] -= __uint_as_float(y.u.y & 0xffff0000u);
            }
        }
    }
}
__device__ __forceinline__ void scaled_parts(const Frag<float>& b, const float* w, Frag<float>* part) {
#pragma unroll
    for (int i = 0; i < 8; i++) part[0].v[i] = w[i] * b.v[i];
}
template <class T> constexpr int kParts = 1;
template <> inline constexpr int kParts<bf16> = 3;

}  // namespace mo
