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
    typedef mo::Tile<T, P> Rows;      // a chunk of q, k, v, ..
    typedef mo::Tile<T, L> Scores;
    static constexpr int STEP = NT / Rows::PIECES, RV = L / STEP;   // rows that the workgroup brings at a time, and times
    static constexpr int TILES = LT == 4 ? 12 : 4;            // score tiles up to the diagonal's 32-blocks
    static constexpr int TPW = (TILES + WAVES - 1) / WAVES;   // a wave's
    static_assert(RV == 2 && STEP % 8 == 0, "");

    static __device__ __forceinline__ void score_tile(int idx, int& it, int& jt) {
        if (LT == 2 || idx < 4) { it = idx >> 1; jt = idx & 1; }
        else { it = 2 + ((idx - 4) >> 2); jt = (idx - 4) & 3; }
    }
};

// What a thread brings of one operand's chunk: a 16-byte piece of row `row` and of the one STEP further, straight into LDS.
// Pieces past the chunk's end or the head's size are zeros (these go through registers).
template <class T, int P> struct Bring {
    typedef Chunk<T, P> C;
    typedef typename C::Rows Rows;
    const T* p;
    int64_t st;
    int col;                   // P where the head ends before the piece
    bool whole;                // the head fills the rows
    __device__ __forceinline__ Bring(const MoRows& r, int64_t n, int h, int d) {
        const int row = threadIdx.x / Rows::PIECES;
        col = ((int)(threadIdx.x % Rows::PIECES) ^ Rows::turn(row)) * C::Rows::EPV;
        st = r.st;
        p = (const T*)r.p + n * r.sn + h * r.sh + row * st + col;
        whole = d == P;
        if (col >= d) col = P;
    }
    __device__ __forceinline__ void chunk(T* tile, int64_t t0, int n) const {
        const T* from = p + t0 * st;
        if (whole && n == C::L) {
            // (a wave's 64 pieces land one after another from the address of its first)
            T* to = tile + threadIdx.x / kWave * (kWave * Rows::EPV);
            typedef __attribute__((address_space(3))) void* Lds;
            typedef const __attribute__((address_space(1))) void* Global;
#pragma unroll
            for (int i = 0; i < C::RV; i++)
                __builtin_amdgcn_global_load_lds((Global)(from + i * C::STEP * st), (Lds)(to + i * C::NT * Rows::EPV), 16, 0, 0);
            return;
        }
        const int row = threadIdx.x / Rows::PIECES;
        uint4 x[C::RV];
#pragma unroll
        for (int i = 0; i < C::RV; i++) {
            x[i] = uint4{0, 0, 0, 0};
            if (row + i * C::STEP < n && col < P) x[i] = *(const uint4*)(from + i * C::STEP * st);
        }
#pragma unroll
        for (int i = 0; i < C::RV; i++) *(uint4*)(tile + ((int)threadIdx.x + i * C::NT) * Rows::EPV) = x[i];
    }
};

// What the workgroup brought is there, for all of it.
__device__ __forceinline__ void brought() {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
}

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

// MODE: KEEP_STATES leaves the states that enter chunks 1, 2, .. for the gradient in a.saved, (N H, chunks - 1, P, P) in the
// elements' type: there they are operands only. ONLY_SUMS makes a segment's own sum.
// A wave's 16 columns (from x0) of a head's (D, E) matrix, or of its transpose, as accumulator tiles.
template <class T, int P, bool TRANSPOSED, class F> __device__ __forceinline__ void each_of_state(const MoAttend& a, int x0, F f) {
    const int lane = threadIdx.x % kWave, g = lane / 16, x = x0 + lane % 16;
    if (a.D == P && a.E == P) {
#pragma unroll
        for (int t = 0; t < P / 16; t++)
#pragma unroll
            for (int r = 0; r < 4; r++) f(t, r, TRANSPOSED ? x * P + acc_row(t, g, r) : acc_row(t, g, r) * P + x);
        return;
    }
#pragma unroll
    for (int t = 0; t < P / 16; t++)
#pragma unroll
        for (int r = 0; r < 4; r++) {
            const int y = acc_row(t, g, r), d = TRANSPOSED ? x : y, e = TRANSPOSED ? y : x;
            if (d < a.D && e < a.E) f(t, r, d * a.E + e);
        }
}

// Where a step does not see another, their product's factor is 0; but 0 times a NaN or an infinity is a NaN, which would reach
// steps of other episodes. Such a value shows in every sum that it entered, so sums that are not finite are made again over
// what is seen only, one product after another. (`none` collects 0 times each sum: a NaN, or 0.)
__device__ __forceinline__ void watch(float& none, const f32x4& x) {
#pragma unroll
    for (int r = 0; r < 4; r++) none = fmaf(x[r], 0.f, none);
}
__device__ __forceinline__ bool any_not_finite(float none) { return __ballot(none != none) != 0; }

template <class T, int P, int MODE>
__global__ void __launch_bounds__((Chunk<T, P>::NT), 4) k_attend(MoAttend a, Cut cut) {
    typedef Chunk<T, P> C;
    constexpr int L = C::L;
    constexpr bool OUT = MODE != ONLY_SUMS;
    __shared__ __align__(16) T lk[L * P], lv[L * P], lq[OUT ? L * P : 8], lp[OUT ? L * L : 8];
    __shared__ float pw[L + 1];
    __shared__ __align__(16) float wt[L];
    const typename C::Rows sk{lk}, sv{lv}, sq{lq};
    const typename C::Scores sp{lp};
    const int w = threadIdx.x / kWave;
    const int64_t nh = blockIdx.x, env = nh / a.H;
    const int h = (int)(nh % a.H), seg = blockIdx.y;
    const int64_t c0 = seg * cut.per_seg, c1 = min(c0 + cut.per_seg, cut.chunks);
    const int e0 = w * 16;     // the wave's columns
    const bool wide_out = rows_wide(a.out, 4 * sizeof(T));
    const int64_t de = (int64_t)a.D * a.E;
    const Bring<T, P> k(a.k, env, h, a.D), v(a.v, env, h, a.E), q(a.q, env, h, a.D);

    f32x4 S[C::PT];
#pragma unroll
    for (int dt = 0; dt < C::PT; dt++) S[dt] = f32x4{0.f, 0.f, 0.f, 0.f};
    const float* in = !OUT ? nullptr : cut.segs > 1 ? cut.enter + ((int64_t)seg * a.N * a.H + nh) * de : a.state ? a.state + nh * de : nullptr;
    if (in) each_of_state<T, P, false>(a, e0, [&](int t, int r, int at) { S[t][r] = in[at]; });
    powers<L>(pw, a.decay[h]);
    bool any_start = false;
    for (int64_t c = c0; c < c1; c++) {
        const int64_t t0 = c * L;
        const int n = (int)min((int64_t)L, a.T - t0);
        __syncthreads();                                       // the last chunk's tiles are done with
        k.chunk(lk, t0, n);
        v.chunk(lv, t0, n);
        if (OUT) q.chunk(lq, t0, n);
        const uint64_t m = __ballot(start_of_lane(a, t0, n, env) != 0);   // the chunk's starts as bits
        any_start |= m != 0;
        const int last = seen_from(m, L - 1);
        if (threadIdx.x < L) wt[threadIdx.x] = (int)threadIdx.x < n && (int)threadIdx.x >= last ? pw[n - 1 - (int)threadIdx.x] : 0.f;
        brought();
        const int lane = lane_here(), g = lane / 16, i16 = lane % 16;

        if (OUT) {
            // scores, transposed: a lane has four neighbouring j of one i
#pragma unroll
            for (int x = 0; x < C::TPW; x++) {
                const int idx = w + x * C::WAVES;
                if (C::TILES % C::WAVES && idx >= C::TILES) break;
                int it, jt;
                C::score_tile(idx, it, jt);
                f32x4 s = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int b = 0; b < C::PB; b++) mma(s, sk.along(jt * 16, b * 32, lane), sq.along(it * 16, b * 32, lane));
                const int i = it * 16 + i16, j = jt * 16 + 4 * g, from = m ? seen_from(m, i) : -1;
                Pack<T, 4> p;
#pragma unroll
                for (int r = 0; r < 4; r++) {
                    const float f = pw[max(i - j - r, 0)];
                    p.v[r] = as<T>(j + r <= i && j + r >= from ? s[r] * f : 0.f);
                }
                *(Pack<T, 4>*)sp.at(i, j) = p;
            }
            if (MODE == KEEP_STATES && c > 0) {                // by rows d, a lane four neighbouring columns
                T* to = (T*)a.saved + (nh * (cut.chunks - 1) + c - 1) * (P * P) + i16 * P + e0 + 4 * g;
#pragma unroll
                for (int t = 0; t < C::PT; t++) {
                    f32x4 x = {0.f, 0.f, 0.f, 0.f};
                    mma(x, frag_of<T>(S[t & ~1], S[t | 1]), unit_frag<T>(t & 1, lane));
                    Pack<T, 4> y;
#pragma unroll
                    for (int r = 0; r < 4; r++) y.v[r] = as<T>(x[r]);
                    *(Pack<T, 4>*)(to + t * 16 * P) = y;
                }
            }
            __syncthreads();
        }

        Frag<T> vf[C::LB];
#pragma unroll
        for (int b = 0; b < C::LB; b++) vf[b] = sv.down(b * 32, e0, lane);

        if (OUT) {
            // outputs, transposed: a lane has four neighbouring columns of one step
            T* out = (T*)a.out.p + env * a.out.sn + h * a.out.sh + e0 + 4 * g + (t0 + i16) * a.out.st;
            const auto write = [&](int it, const f32x4& own, const f32x4& far) {
                const int i = it * 16 + i16;
                const bool enters = !m || seen_from(m, i) < 0;
                const float f = pw[i + 1];
                Pack<T, 4> y;
#pragma unroll
                for (int r = 0; r < 4; r++) y.v[r] = as<T>(a.scale * (enters ? fmaf(f, far[r], own[r]) : own[r]));
                if (i < n && e0 + 4 * g < a.E) put4(out + it * 16 * a.out.st, y, wide_out);
            };
            Frag<T> sf[C::PB];
#pragma unroll
            for (int b = 0; b < C::PB; b++) sf[b] = frag_of<T>(S[2 * b], S[2 * b + 1]);
            float none = 0.f;
#pragma unroll
            for (int it = 0; it < C::LT; it++) {
                f32x4 own = {0.f, 0.f, 0.f, 0.f}, far = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int b = 0; b < C::PB; b++) mma(far, sf[b], sq.along(it * 16, b * 32, lane));
#pragma unroll
                for (int b = 0; b <= it / 2; b++) mma(own, vf[b], sp.along(it * 16, b * 32, lane));
                watch(none, own);
                write(it, own, far);
            }
            if (any_not_finite(none)) {
#pragma unroll 1
                for (int it = 0; it < C::LT; it++) {
                    const int i = it * 16 + i16;
                    f32x4 own = {0.f, 0.f, 0.f, 0.f}, far = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int b = 0; b < C::PB; b++) mma(far, sf[b], sq.along(it * 16, b * 32, lane));
#pragma unroll 1
                    for (int j = max(seen_from(m, i), 0); j <= i; j++)
#pragma unroll
                        for (int r = 0; r < 4; r++) own[r] = fmaf(as_f32(*sp.at(i, j)), as_f32(*sv.at(j, e0 + 4 * g + r)), own[r]);
                    write(it, own, far);
                }
            }
        }

        f32x4 add[C::PT];
#pragma unroll
        for (int dt = 0; dt < C::PT; dt++) add[dt] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int b = 0; b < C::LB; b++) {
            Frag<T> part[kParts<T>];
            scaled_parts(vf[b], &wt[b * 32 + 8 * g], part);
#pragma unroll
            for (int dt = 0; dt < C::PT; dt++) {
                const Frag<T> kf = sk.template down<true>(b * 32, acc_col(dt), lane);
#pragma unroll
                for (int p = 0; p < kParts<T>; p++) mma(add[dt], kf, part[p]);
            }
        }
        float none = 0.f;
#pragma unroll
        for (int dt = 0; dt < C::PT; dt++) watch(none, add[dt]);
        if (any_not_finite(none)) {
#pragma unroll
            for (int dt = 0; dt < C::PT; dt++) {
                add[dt] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll 1
                for (int j = max(last, 0); j < n; j++)
#pragma unroll
                    for (int r = 0; r < 4; r++)
                        add[dt][r] = fmaf(wt[j] * as_f32(*sk.at(j, acc_row(dt, g, r))), as_f32(*sv.at(j, e0 + i16)), add[dt][r]);
            }
        }
        const float f = pw[n];
#pragma unroll
        for (int dt = 0; dt < C::PT; dt++)
#pragma unroll
            for (int r = 0; r < 4; r++) S[dt][r] = last < 0 ? fmaf(f, S[dt][r], add[dt][r]) : add[dt][r];
    }
    float* to = !OUT ? cut.enter + ((int64_t)seg * a.N * a.H + nh) * de : cut.segs > 1 ? nullptr : a.state_out + nh * de;
    if (to) each_of_state<T, P, false>(a, e0, [&](int t, int r, int at) { to[at] = S[t][r]; });
    if (!OUT && threadIdx.x == 0) {
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
inline int64_t saved_bytes(const MoAttend& a) {
    const int64_t p = padded_head(a);
    return a.N * a.H * ((a.T + chunk_steps(a) - 1) / chunk_steps(a) - 1) * p * p * (a.dtype == MO_BF16 ? 2 : 4);
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
