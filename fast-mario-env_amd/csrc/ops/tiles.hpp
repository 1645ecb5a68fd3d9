// 16 x 16 matrix-instruction tiles whose operands lie in LDS, for bf16 (one 16x16x32 product) and float32 (eight 16x16x4).
#pragma once
#include "common.hpp"

namespace mo {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef short i16x4 __attribute__((ext_vector_type(4)));
typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));

// An operand of a product over 32 indices: lane l has row (of A) or column (of B) l % 16 and eight of the indices. Which eight
// is up to the caller, as long as A and B agree: 8 (l / 16) + 0..7 ("in order"), or 4 (l / 16) + 0..3 and the same + 16
// ("in halves"): the rows that a lane holds of two stacked accumulator tiles, so that an accumulator becomes an operand in place.
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

// p: row l % 16 of the operand at its first index; the lane's eight indices in order or in halves.
__device__ __forceinline__ Frag<bf16> frag_in_order(const bf16* p, int g) { return {*(const bf16x8*)(p + 8 * g)}; }
__device__ __forceinline__ Frag<float> frag_in_order(const float* p, int g) {
    Frag<float> f;
    *(f32x4*)f.v = *(const f32x4*)(p + 8 * g);
    *(f32x4*)(f.v + 4) = *(const f32x4*)(p + 8 * g + 4);
    return f;
}
__device__ __forceinline__ Frag<bf16> frag_in_halves(const bf16* p, int g) {
    const bf16x4 a = *(const bf16x4*)(p + 4 * g), b = *(const bf16x4*)(p + 16 + 4 * g);
    return {__builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7)};
}
__device__ __forceinline__ Frag<float> frag_in_halves(const float* p, int g) {
    Frag<float> f;
    *(f32x4*)f.v = *(const f32x4*)(p + 4 * g);
    *(f32x4*)(f.v + 4) = *(const f32x4*)(p + 16 + 4 * g);
    return f;
}

// The operand whose indices run down the rows of a tile: p its first row at the operand's first row or column, ld its row
// stride. In order. bf16 takes the transposing LDS read: 16 lanes read 4 rows of 16 and each gets a column.
__device__ __forceinline__ Frag<bf16> frag_down(const bf16* p, int ld, int lane) {
    typedef __attribute__((address_space(3))) i16x4* Lds;
    const int g = lane / 16, i = lane % 16;
    const bf16* q = p + (8 * g + i / 4) * ld + (i % 4) * 4;
    union { i16x4 h[2]; Frag<bf16> f; } u;
    u.h[0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((Lds)q);
    u.h[1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((Lds)(q + 4 * ld));
    return u.f;
}
__device__ __forceinline__ Frag<float> frag_down(const float* p, int ld, int lane) {
    const float* q = p + 8 * (lane / 16) * ld + lane % 16;
    Frag<float> f;
#pragma unroll
    for (int i = 0; i < 8; i++) f.v[i] = q[i * ld];
    return f;
}

// Two stacked accumulator tiles as an operand, indices in halves: the one rounding of what they hold.
__device__ __forceinline__ Frag<bf16> frag_of(const f32x4& a, const f32x4& b) {
    Frag<bf16> f;
#pragma unroll
    for (int i = 0; i < 4; i++) { f.v[i] = (bf16)a[i]; f.v[4 + i] = (bf16)b[i]; }
    return f;
}
__device__ __forceinline__ Frag<float> frag_of_f32(const f32x4& a, const f32x4& b) {
    Frag<float> f;
#pragma unroll
    for (int i = 0; i < 4; i++) { f.v[i] = a[i]; f.v[4 + i] = b[i]; }
    return f;
}
template <class T> __device__ __forceinline__ Frag<T> state_frag(const f32x4& a, const f32x4& b);
template <> __device__ __forceinline__ Frag<bf16> state_frag<bf16>(const f32x4& a, const f32x4& b) { return frag_of(a, b); }
template <> __device__ __forceinline__ Frag<float> state_frag<float>(const f32x4& a, const f32x4& b) { return frag_of_f32(a, b); }

// acc += A (w B), w a factor for each index, with float32's precision: w B is split into bf16 parts of 8 bits of significand
// each, three of which leave 2^-27 of it. (Where w is 0 the value is left out, whatever it is.)
__device__ __forceinline__ void scaled_parts(const Frag<bf16>& b, const float* w, Frag<bf16>* part) {
#pragma unroll
    for (int i = 0; i < 8; i++) {
        float x = w[i] == 0.f ? 0.f : w[i] * (float)b.v[i];
#pragma unroll
        for (int p = 0; p < 3; p++) {
            part[p].v[i] = (bf16)x;
            x -= (float)part[p].v[i];
        }
    }
}
__device__ __forceinline__ void scaled_parts(const Frag<float>& b, const float* w, Frag<float>* part) {
#pragma unroll
    for (int i = 0; i < 8; i++) part[0].v[i] = w[i] == 0.f ? 0.f : w[i] * b.v[i];
}
template <class T> constexpr int kParts = 1;
template <> inline constexpr int kParts<bf16> = 3;

// Whether any of the 16 bytes' values is infinite or a NaN: the largest magnitude's bits so far, and what they say.
__device__ __forceinline__ uint32_t most_bits(uint32_t most, const uint4& x, bf16) {
    union { uint32_t u; u16x2 h; } m{most};
    for (uint32_t w : {x.x, x.y, x.z, x.w}) {
        union { uint32_t u; u16x2 h; } y{w & 0x7fff7fffu};
        m.h = __builtin_elementwise_max(m.h, y.h);
    }
    return m.u;
}
__device__ __forceinline__ uint32_t most_bits(uint32_t most, const uint4& x, float) {
    for (uint32_t w : {x.x, x.y, x.z, x.w}) most = max(most, w & 0x7fffffffu);
    return most;
}
__device__ __forceinline__ bool not_finite(uint32_t most, bf16) { return (most >> 16) >= 0x7f80u || (most & 0xffffu) >= 0x7f80u; }
__device__ __forceinline__ bool not_finite(uint32_t most, float) { return most >= 0x7f800000u; }

}  // namespace mo
