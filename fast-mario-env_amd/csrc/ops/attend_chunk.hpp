// Linear attention by chunks of steps on the matrix cores: the forward pass.
#pragma once
#include "tiles.hpp"

namespace mo {

// A chunk is L steps. With S the state that enters it, G_ij = g^(i-j) where step i sees step j (j <= i and no episode starts
// in j + 1 .. i) and else 0:
//   O  = scale ((Q K^T . G) V + diag(g^(i+1), 0 past the first start) Q S)
//   S' = (no start in the chunk ? g^n : 0) S + K^T diag(w) V,   w_j = g^(n-1-j), 0 before the last start
// A workgroup takes one env's head and walks its chunks (or a cut of them) with S in registers: wave w holds the 16 columns
// of S from 16 w, all rows, as accumulator tiles, which are the operand of Q S as they lie. Everything is read once and
// written once; a chunk is three products over 32-step blocks of at most L x L x P, far below what the matrix cores do in the
// time its rows take to come, so the pass is bound by memory as long as enough workgroups wait for it at once.
//
// T: element type. P: head size rounded up to 32, 64 or 128; columns past D or E are zeros. L: 64 for bf16; 32 for float32,
// whose matrix instructions are 16 times slower, so that the products of a chunk with itself stay short.
template <class T, int P> struct Chunk {
    static constexpr int L = sizeof(T) == 2 ? 64 : 32;
    static constexpr int WAVES = P / 16, NT = WAVES * kWave;
    static constexpr int LT = L / 16, LB = L / 32, PB = P / 32, PT = P / 16;
    static constexpr int PAD = 16 / sizeof(T), LD = P + PAD, LS = L + PAD;    // LDS row strides: 16 bytes past a power of two
    static constexpr int EPV = 16 / sizeof(T), VPR = P / EPV, RV = L * VPR / NT;   // 16-byte accesses: a row's, a thread's
    static constexpr int TILES = LT == 4 ? 12 : 4;                            // score tiles up to the diagonal's 32-blocks
    static_assert(RV == 2 && L * VPR % NT == 0, "");
    typedef T Tile[L][LD];

    static __device__ __forceinline__ void score_tile(int idx, int& it, int& jt) {
        if (LT == 2 || idx < 4) { it = idx >> 1; jt = idx & 1; }
        else { it = 2 + ((idx - 4) >> 2); jt = (idx - 4) & 3; }
    }
};

// What a thread brings of one operand's tile: its 16-byte pieces, of which pieces past the chunk's end or the head's size
// are zeros.
template <class T, int P> struct Rows {
    typedef Chunk<T, P> C;
    const T* p[C::RV];
    int64_t st;
    int row[C::RV], col;
    uint4 x[C::RV];
    __device__ __forceinline__ void init(const MoRows& r, int64_t n, int h, int d) {
        st = r.st;
        col = (int)(threadIdx.x % C::VPR) * C::EPV;
#pragma unroll
        for (int i = 0; i < C::RV; i++) {
            row[i] = (int)threadIdx.x / C::VPR + i * (C::NT / C::VPR);
            p[i] = (const T*)r.p + n * r.sn + h * r.sh + row[i] * r.st + col;
            if (col >= d) row[i] = C::L;
        }
    }
    __device__ __forceinline__ void load(int64_t t0, int n) {
#pragma unroll
        for (int i = 0; i < C::RV; i++) {
            x[i] = uint4{0, 0, 0, 0};
            if (row[i] < n) x[i] = *(const uint4*)(p[i] + t0 * st);
        }
    }
    __device__ __forceinline__ void put(T (*tile)[C::LD]) {
#pragma unroll
        for (int i = 0; i < C::RV; i++)
            *(uint4*)&tile[(int)threadIdx.x / C::VPR + i * (C::NT / C::VPR)][col] = x[i];
    }
    __device__ __forceinline__ uint32_t most(uint32_t m) const {
#pragma unroll
        for (int i = 0; i < C::RV; i++) m = most_bits(m, x[i], T{});
        return m;
    }
};

// Four neighbouring values, in one access where the rows allow it.
__device__ __forceinline__ bool rows_wide(const MoRows& r, size_t bytes) {
    return ((uintptr_t)r.p % bytes == 0) & ((uint64_t)(r.st | r.sn | r.sh) % 4 == 0);
}
template <class T> __device__ __forceinline__ void put4(T* p, const Pack<T, 4>& y, bool wide) {
    if (wide) *(Pack<T, 4>*)p = y;
    else
#pragma unroll
        for (int r = 0; r < 4; r++) p[r] = y.v[r];
}

// The latest start at or before step i of a chunk whose starts are the bits of m, or -1: step i sees the steps from there on.
__device__ __forceinline__ int seen_from(uint64_t m, int i) {
    const uint64_t low = m & (~0ull >> (63 - i));
    return 63 - __clzll((long long)low);   // (__clzll(0) is 64)
}

// Whether step t0 + (the lane's number) of the n from t0 starts an episode.
__device__ __forceinline__ int start_of_lane(const MoAttend& a, int64_t t0, int n, int64_t env) {
    const int lane = threadIdx.x % kWave;
    return a.start && lane < n ? a.start[(t0 + lane) * a.N + env] : 0;
}

// g^0 .. g^L. (g^0 is 1 for g = 0 too.)
template <int L> __device__ __forceinline__ void powers(float* pw, float g) {
    const float lg = __log2f(g);
    for (int i = threadIdx.x; i <= L; i += blockDim.x) pw[i] = i ? exp2f((float)i * lg) : 1.f;
}

// A long sequence is cut into segments of whole chunks, a workgroup each, so that few sequences fill the chip. First each
// segment's own sum and what it leaves of an entering state (`keep`: g^steps, or -1 where an episode starts inside), then the
// states that enter the segments one after another, then the outputs from there.
struct Cut {
    int64_t chunks, per_seg;   // chunks of a sequence and of a segment
    int segs;
    float* enter;              // (segs, N H, D E): a segment's own sum, then the state that enters it
    float* keep;               // (segs, N H)
};

enum { KEEP_NONE = 0, KEEP_STATES = 1, ONLY_SUMS = 2 };

// MODE: KEEP_STATES leaves the states that enter chunks 1, 2, .. for the gradient in a.saved, (N H, chunks - 1, D, E) in the
// elements' type: there they are operands only. ONLY_SUMS makes a segment's own sum.
template <class T, int P, int MODE>
__global__ void __launch_bounds__((Chunk<T, P>::NT)) k_attend(MoAttend a, Cut cut) {
    typedef Chunk<T, P> C;
    constexpr int L = C::L;
    __shared__ __align__(16) T sk[L][C::LD], sv[L][C::LD];
    __shared__ __align__(16) T sq[MODE == ONLY_SUMS ? 1 : L][C::LD], sp[MODE == ONLY_SUMS ? 1 : L][C::LS];
    __shared__ float pw[L + 1];
    __shared__ __align__(16) float wt[L];
    __shared__ int odd[2];     // a value that is not finite is in the chunk's k or v
    const int lane = threadIdx.x % kWave, w = threadIdx.x / kWave, g = lane / 16, i16 = lane % 16;
    const int64_t nh = blockIdx.x, env = nh / a.H;
    const int h = (int)(nh % a.H), seg = blockIdx.y;
    const int64_t c0 = seg * cut.per_seg, c1 = min(c0 + cut.per_seg, cut.chunks);
    const int e0 = w * 16;     // the wave's columns
    const bool wide_out = rows_wide(a.out, 4 * sizeof(T));
    const int64_t de = (int64_t)a.D * a.E;

    powers<L>(pw, a.decay[h]);
    if (threadIdx.x < 2) odd[threadIdx.x] = 0;
    f32x4 S[C::PT];
    const float* in = MODE == ONLY_SUMS ? nullptr : cut.segs > 1 ? cut.enter + ((int64_t)seg * a.N * a.H + nh) * de : a.state ? a.state + nh * de : nullptr;
#pragma unroll
    for (int dt = 0; dt < C::PT; dt++)
#pragma unroll
        for (int r = 0; r < 4; r++) {
            const int d = dt * 16 + 4 * g + r, e = e0 + i16;
            S[dt][r] = in && d < a.D && e < a.E ? in[d * a.E + e] : 0.f;
        }
    Rows<T, P> q, k, v;
    k.init(a.k, env, h, a.D);
    v.init(a.v, env, h, a.E);
    if (MODE != ONLY_SUMS) q.init(a.q, env, h, a.D);
    const auto steps = [&](int64_t c) { return (int)min((int64_t)L, a.T - c * L); };
    int starts = 0;
    const auto fetch = [&](int64_t c) {
        starts = start_of_lane(a, c * L, steps(c), env);
        k.load(c * L, steps(c));
        v.load(c * L, steps(c));
        if (MODE != ONLY_SUMS) q.load(c * L, steps(c));
    };
    if (c0 < c1) fetch(c0);
    bool any_start = false;
    for (int64_t c = c0; c < c1; c++) {
        const int n = steps(c);
        const int64_t t0 = c * L;
        __syncthreads();                                       // the last chunk's tiles are done with
        k.put(sk);
        v.put(sv);
        if (MODE != ONLY_SUMS) q.put(sq);
        const uint64_t m = __ballot(starts != 0);   // the chunk's starts as bits
        any_start |= m != 0;
        const int last = seen_from(m, L - 1);
        if (threadIdx.x < L) wt[threadIdx.x] = (int)threadIdx.x < n && (int)threadIdx.x >= last ? pw[n - 1 - (int)threadIdx.x] : 0.f;
        if (not_finite(v.most(k.most(0)), T{})) odd[c & 1] = 1;
        __syncthreads();
        if (c + 1 < c1) fetch(c + 1);
        const bool exact_sums = odd[c & 1];
        if (threadIdx.x == 0) odd[(c + 1) & 1] = 0;

        if (MODE != ONLY_SUMS) {
            // scores, transposed: a lane has four neighbouring j of one i
            for (int idx = w; idx < C::TILES; idx += C::WAVES) {
                int it, jt;
                C::score_tile(idx, it, jt);
                f32x4 s = {0.f, 0.f, 0.f, 0.f};
                if (jt <= it) {
#pragma unroll
                    for (int b = 0; b < C::PB; b++)
                        mma(s, frag_in_order(&sk[jt * 16 + i16][b * 32], g), frag_in_order(&sq[it * 16 + i16][b * 32], g));
                    const int i = it * 16 + i16, j = jt * 16 + 4 * g, from = seen_from(m, i);
#pragma unroll
                    for (int r = 0; r < 4; r++) s[r] = j + r <= i && j + r >= from ? s[r] * pw[max(i - j - r, 0)] : 0.f;
                }
                Pack<T, 4> p;
#pragma unroll
                for (int r = 0; r < 4; r++) p.v[r] = as<T>(s[r]);
                *(Pack<T, 4>*)&sp[it * 16 + i16][jt * 16 + 4 * g] = p;
            }
            if (MODE == KEEP_STATES && c > 0) {
                T* to = (T*)a.saved + (nh * (cut.chunks - 1) + c - 1) * de;
#pragma unroll
                for (int dt = 0; dt < C::PT; dt++)
#pragma unroll
                    for (int r = 0; r < 4; r++) {
                        const int d = dt * 16 + 4 * g + r, e = e0 + i16;
                        if (d < a.D && e < a.E) to[d * a.E + e] = as<T>(S[dt][r]);
                    }
            }
            __syncthreads();
        }

        Frag<T> vf[C::LB];
#pragma unroll
        for (int b = 0; b < C::LB; b++) vf[b] = frag_down(&sv[b * 32][e0], C::LD, lane);

        if (MODE != ONLY_SUMS) {
            // outputs, transposed: a lane has four neighbouring columns of one step
            f32x4 o[C::LT], x[C::LT];
#pragma unroll
            for (int it = 0; it < C::LT; it++) {
                o[it] = f32x4{0.f, 0.f, 0.f, 0.f};
                x[it] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int b = 0; b <= it / 2; b++)
                    if (!exact_sums) mma(o[it], vf[b], frag_in_order(&sp[it * 16 + i16][b * 32], g));
            }
            if (exact_sums) {                                  // 0 times a NaN that a step must not see would be one
#pragma unroll
                for (int it = 0; it < C::LT; it++) {
                    const int i = it * 16 + i16;
                    for (int j = max(seen_from(m, i), 0); j <= i; j++)
#pragma unroll
                        for (int r = 0; r < 4; r++) o[it][r] = fmaf(as_f32(sp[i][j]), as_f32(sv[j][e0 + 4 * g + r]), o[it][r]);
                }
            }
#pragma unroll
            for (int b = 0; b < C::PB; b++) {
                const Frag<T> sf = state_frag<T>(S[2 * b], S[2 * b + 1]);
#pragma unroll
                for (int it = 0; it < C::LT; it++) mma(x[it], sf, frag_in_halves(&sq[it * 16 + i16][b * 32], g));
            }
            T* out = (T*)a.out.p + env * a.out.sn + h * a.out.sh + e0 + 4 * g;
#pragma unroll
            for (int it = 0; it < C::LT; it++) {
                const int i = it * 16 + i16;
                if (i >= n || e0 + 4 * g >= a.E) continue;
                const bool enters = seen_from(m, i) < 0;
                const float f = pw[i + 1];
                Pack<T, 4> y;
#pragma unroll
                for (int r = 0; r < 4; r++) y.v[r] = as<T>(a.scale * (enters ? fmaf(f, x[it][r], o[it][r]) : o[it][r]));
                put4(out + (t0 + i) * a.out.st, y, wide_out);
            }
        }

        const float f = last < 0 ? pw[n] : 0.f;
        if (!exact_sums) {
            Frag<T> part[C::LB][kParts<T>];
#pragma unroll
            for (int b = 0; b < C::LB; b++) scaled_parts(vf[b], &wt[b * 32 + 8 * g], part[b]);
#pragma unroll
            for (int dt = 0; dt < C::PT; dt++) {
#pragma unroll
                for (int r = 0; r < 4; r++) S[dt][r] = last < 0 ? f * S[dt][r] : 0.f;
#pragma unroll
                for (int b = 0; b < C::LB; b++) {
                    const Frag<T> kf = frag_down(&sk[b * 32][dt * 16], C::LD, lane);
#pragma unroll
                    for (int p = 0; p < kParts<T>; p++) mma(S[dt], kf, part[b][p]);
                }
            }
        } else {
#pragma unroll
            for (int dt = 0; dt < C::PT; dt++)
#pragma unroll
                for (int r = 0; r < 4; r++) {
                    float s = last < 0 ? f * S[dt][r] : 0.f;
                    for (int j = max(last, 0); j < n; j++) s = fmaf(wt[j] * as_f32(sk[j][dt * 16 + 4 * g + r]), as_f32(sv[j][e0 + i16]), s);
                    S[dt][r] = s;
                }
        }
    }
    float* to = MODE == ONLY_SUMS ? cut.enter + ((int64_t)seg * a.N * a.H + nh) * de : cut.segs > 1 ? nullptr : a.state_out + nh * de;
    if (to)
#pragma unroll
        for (int dt = 0; dt < C::PT; dt++)
#pragma unroll
            for (int r = 0; r < 4; r++) {
                const int d = dt * 16 + 4 * g + r, e = e0 + i16;
                if (d < a.D && e < a.E) to[d * a.E + e] = S[dt][r];
            }
    if (MODE == ONLY_SUMS && threadIdx.x == 0) {
        const int64_t n = min(c1 * L, a.T) - c0 * L;
        cut.keep[(int64_t)seg * a.N * a.H + nh] = any_start ? -1.f : exp2f((float)n * __log2f(a.decay[h]));
    }
}

// The states that enter the segments, in place of the segments' sums, and the last one: a thread an element, over the segments
// in order (forwards or backwards).
struct Enter {
    float* enter;
    const float* keep;
    const float* first;        // null: zeros
    float* last;               // null: not wanted
    int64_t elements, de, nh;  // of all states; of one; number of them
    int segs;
    bool back;
};
__global__ void __launch_bounds__(256) k_attend_enter(Enter k) {
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= k.elements) return;
    const int64_t nh = i / k.de;
    float S = k.first ? k.first[i] : 0.f;
    for (int s0 = 0; s0 < k.segs; s0 += 8) {
        float own[8], keep[8];
#pragma unroll
        for (int j = 0; j < 8; j++)
            if (s0 + j < k.segs) {
                const int s = k.back ? k.segs - 1 - (s0 + j) : s0 + j;
                own[j] = k.enter[s * k.elements + i];
                keep[j] = k.keep[s * k.nh + nh];
            }
#pragma unroll
        for (int j = 0; j < 8; j++)
            if (s0 + j < k.segs) {
                const int s = k.back ? k.segs - 1 - (s0 + j) : s0 + j;
                k.enter[s * k.elements + i] = S;
                S = keep[j] < 0.f ? own[j] : fmaf(keep[j], S, own[j]);
            }
    }
    if (k.last) k.last[i] = S;
}

// ---- host side
inline bool rows_suit(const MoRows& r, int64_t epv) {   // 16-byte accesses
    return (uintptr_t)r.p % 16 == 0 && r.st % epv == 0 && r.sn % epv == 0 && r.sh % epv == 0;
}
// The chunk kernels take heads of whole 16-byte pieces whose rows lie on them; the rest goes step by step (k_walk).
inline bool chunks_take(const MoAttend& a, bool backward) {
    const int64_t epv = a.dtype == MO_BF16 ? 8 : 4;
    if (a.T == 0 || a.D % epv || a.E % epv || !rows_suit(a.q, epv) || !rows_suit(a.k, epv) || !rows_suit(a.v, epv)) return false;
    return !backward || rows_suit(a.dout, epv);
}
inline int chunk_steps(const MoAttend& a) { return a.dtype == MO_BF16 ? 64 : 32; }
inline int padded_head(const MoAttend& a) { const int m = std::max(a.D, a.E); return m <= 32 ? 32 : m <= 64 ? 64 : 128; }

// Segments: where the sequences alone would leave compute units without `per_cu` workgroups.
inline Cut attend_cut(const MoAttend& a, int per_cu) {
    Cut c{};
    c.chunks = (a.T + chunk_steps(a) - 1) / chunk_steps(a);
    const int64_t want = (int64_t)compute_units() * per_cu / std::max<int64_t>(1, a.N * a.H);
    const int64_t segs = std::max<int64_t>(1, std::min(want, c.chunks / 2));
    c.per_seg = std::max<int64_t>(1, (c.chunks + segs - 1) / segs);
    c.segs = (int)std::max<int64_t>(1, (c.chunks + c.per_seg - 1) / c.per_seg);
    return c;
}
inline int64_t cut_bytes(const MoAttend& a, const Cut& c) {
    return c.segs > 1 ? (int64_t)c.segs * a.N * a.H * (4 * (int64_t)a.D * a.E + 4) : 0;
}
inline void cut_place(const MoAttend& a, Cut& c) {
    c.enter = (float*)a.work;
    c.keep = c.enter + (int64_t)c.segs * a.N * a.H * a.D * a.E;
}
inline int enter_states(const MoAttend& a, const Cut& c, const float* first, float* last, bool back, hipStream_t s) {
    const int64_t de = (int64_t)a.D * a.E, nh = a.N * a.H;
    hipLaunchKernelGGL(k_attend_enter, dim3((unsigned)((nh * de + 255) / 256)), dim3(256), 0, s,
                       Enter{c.enter, c.keep, first, last, nh * de, de, nh, c.segs, back});
    return launched("k_attend_enter");
}

constexpr int FORWARD_PER_CU = 4;

template <class T, int P> int attend_chunks(const MoAttend& a, hipStream_t s) {
    Cut c = attend_cut(a, FORWARD_PER_CU);
    cut_place(a, c);
    const dim3 grid((unsigned)(a.N * a.H), (unsigned)c.segs), block(Chunk<T, P>::NT);
    if (c.segs > 1) {
        hipLaunchKernelGGL((k_attend<T, P, ONLY_SUMS>), grid, block, 0, s, a, c);
        if (launched("k_attend sums") || enter_states(a, c, a.state, a.state_out, false, s)) return -1;
    }
    if (a.saved && c.chunks > 1) hipLaunchKernelGGL((k_attend<T, P, KEEP_STATES>), grid, block, 0, s, a, c);
    else hipLaunchKernelGGL((k_attend<T, P, KEEP_NONE>), grid, block, 0, s, a, c);
    return launched("k_attend");
}

}  // namespace mo
