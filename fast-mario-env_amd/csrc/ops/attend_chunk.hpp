// Linear attention by chunks of steps on the matrix cores: the forward pass.
#pragma once
#include "tiles.hpp"

namespace mo {

// A chunk is L steps. With S the state that enters it, G_ij = g^(i-j) where step i sees step j (j <= i and no episode starts
// in j + 1 .. i) and else 0:
//   O  = scale ((Q K^T . G) V + diag(g^(i+1), 0 past the first start) Q S)
//   S' = (no start in the chunk ? g^n : 0) S + K^T diag(w) V,   w_j = g^(n-1-j), 0 before the last start
// A workgroup takes one env's head and walks its chunks (or a cut of them) with S in registers: wave w holds the 16 columns
// of S from 16 w, all rows, as accumulator tiles, which are the operand of Q S as they lie. S and the masked scores go into products in
// two parts (halves, in tiles.hpp), S' is made from w V in three (scaled_parts). Everything is read once and
// written once; a chunk is three products over 32-step blocks of at most L x L x P, far below what the matrix cores do in the
// time its rows take to come, so the pass is bound by memory as long as enough workgroups wait for it at once: three fit a
// compute unit (two of heads of 128, whose 256 registers spill two).
//
// Measured, bf16, D = E = 64 and 8 heads, 128 steps of 4,096 envs: 753 us for 3.2 GB, 4.3 TB/s, where a copy of 1 GiB reaches 5.2; its
// bytes cross once, the matrix units are busy 15 % of the time and waves wait 41 % of theirs (counters). (Step by step, k_walk: 4,889
// us.) From zeros, 2,056 envs: 302 us, 4.5 TB/s (287 with one part of S and scores); 1,000 envs with heads of 128: 371 us, 4.2 TB/s
// (335); with heads of 64 140 us (130), in float32 281.
// Where a step's rows lie a multiple of 2 MiB apart (N H D a power of two), a pass takes longer: from zeros and keeping the states
// for the gradient, 2,048 envs take 385 us, 2,056 take 325.
//
// T: element type. P: head size rounded up to 32, 64 or 128; columns past D or E are zeros. L: 64 for bf16; 32 for float32,
// whose matrix instructions are 16 times slower, so that the products of a chunk with itself stay short.
//
// W: waves of the workgroup.
template <class T, int P, int W> struct Chunk {
    static constexpr int L = sizeof(T) == 2 ? 64 : 32;
    static constexpr int WAVES = W, NT = W * kWave;
    static constexpr int CT = P / 16 / W;                     // 16-column tiles of S of a wave
    static constexpr int LT = L / 16, LB = L / 32, PB = P / 32, PT = P / 16;
    typedef Tile<T, P> Rows;          // a chunk of q, k, v, ..
    typedef ScoreParts<T, L> Scored;
    static constexpr int SCORES = kHalves<T> * Scores<T, L>::SIZE, K = kHalves<T>;
    static constexpr int STEP = NT / Rows::PIECES, RV = L / STEP;   // rows that the workgroup moves at a time, and times
    static constexpr int TILES = LT == 4 ? 12 : 4;            // score tiles up to the diagonal's 32-blocks
    static constexpr int TPW = (TILES + W - 1) / W;           // a wave's
    static_assert(CT * W * 16 == P && RV * STEP == L && STEP % 8 == 0, "");

    static __device__ __forceinline__ void score_tile(int idx, int& it, int& jt) {
        if (LT == 2 || idx < 4) { it = idx >> 1; jt = idx & 1; }
        else { it = 2 + ((idx - 4) >> 2); jt = (idx - 4) & 3; }
    }
};

// The thread's number, not known to be the same from one pass of a loop to the next: what follows from it (addresses, mostly) is
// then made where it is used, instead of being kept in registers over the whole loop, which costs more in waves than it saves.
__device__ __forceinline__ unsigned thread_here() {
    unsigned t = threadIdx.x;
    asm volatile("" : "+v"(t));
    return t;
}

// The rows of one operand or result of an env's head, d wide. A thread moves a 16-byte piece of row t / PIECES and of every
// STEP-th after it.
template <class T, class C> struct HeadRows {
    typedef typename C::Rows Tl;
    T* p;
    int64_t st;
    int d;
    bool whole;                // 16-byte pieces only: the head fills the tile's rows; of a result: its rows lie on 16 bytes
    __device__ __forceinline__ HeadRows(const MoRows& r, int64_t n, int h, int size, bool w) : p((T*)r.p + n * r.sn + h * r.sh), st(r.st), d(size), whole(w) {}

    // Straight into LDS, where a wave's 64 pieces land one after another. (Rows past the chunk's end and columns past the
    // head's size are zeros; such chunks go through registers.)
    __device__ __forceinline__ void bring(T* tile, int64_t t0, int n) const {
        const unsigned t = thread_here(), row = t / Tl::PIECES, col = ((t % Tl::PIECES) ^ Tl::turn(row)) * Tl::EPV;
        const T* from = p + (t0 + row) * st + col;
        if (whole && n == C::L) {
            T* to = tile + threadIdx.x / kWave * (kWave * Tl::EPV);
            typedef __attribute__((address_space(3))) void* Lds;
            typedef const __attribute__((address_space(1))) void* Global;
#pragma unroll
            for (int i = 0; i < C::RV; i++)
                __builtin_amdgcn_global_load_lds((Global)(from + i * C::STEP * st), (Lds)(to + i * C::NT * Tl::EPV), 16, 0, 2 /* nt: read once */);
            return;
        }
#pragma unroll
        for (int i = 0; i < C::RV; i++) {
            uint4 x = {0, 0, 0, 0};
            if ((int)row + i * C::STEP < n && (int)col < d) x = *(const uint4*)(from + i * C::STEP * st);
            *(uint4*)(tile + (t + i * C::NT) * Tl::EPV) = x;
        }
    }

    // Results from LDS. (Straight from the accumulators, four values of each of 16 rows at a time, the stores of the forward
    // pass took longer than its loads and products together.)
    __device__ __forceinline__ void take(const T* tile, int64_t t0, int n) const {
        typedef Pack<T, Tl::EPV> Piece;
        const unsigned t = thread_here(), row = t / Tl::PIECES, col = ((t % Tl::PIECES) ^ Tl::turn(row)) * Tl::EPV;
        T* to = p + (t0 + row) * st + col;
#pragma unroll
        for (int i = 0; i < C::RV; i++) {
            const Piece x = *(const Piece*)(tile + (t + i * C::NT) * Tl::EPV);
            if ((int)row + i * C::STEP >= n || (int)col >= d) continue;
            if (whole) stream((Piece*)(to + i * C::STEP * st), x);
            else
#pragma unroll
                for (int j = 0; j < Tl::EPV; j++) to[i * C::STEP * st + j] = x.v[j];
        }
    }
};
template <class T> __device__ __forceinline__ bool on_pieces(const MoRows& r) {
    return ((uintptr_t)r.p % 16 == 0) & ((uint64_t)(r.st | r.sn | r.sh) % (16 / sizeof(T)) == 0);
}

// What the workgroup brought is there, for all of it.
__device__ __forceinline__ void brought() {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
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

// g^n, 1 for n = 0, rounded once: squares in float64. (A logarithm's rounding would grow with the memory's length: with g = 1 - x
// it enters a state as its error over x.)
__device__ __forceinline__ float power(float g, int64_t n) {
    double p = 1.0;
    for (double x = g; n; n >>= 1, x *= x)
        if (n & 1) p *= x;
    return (float)p;
}

// g^0 .. g^L, and the factors by which step i sees step j, scale g^(i-j) or 0, of all i - j.
template <int L> struct Powers {
    float pw[L + 1], seen[2 * L];
    __device__ __forceinline__ void fill(float g, float scale) {
        for (int i = threadIdx.x; i <= L; i += blockDim.x) {
            const float x = power(g, i);
            pw[i] = x;
            if (i < L) { seen[i] = 0.f; seen[L + i] = scale * x; }
        }
    }
    __device__ __forceinline__ const float* sees(int i, int j) const { return &seen[L + i - j]; }
};

// The env and head of a workgroup. Workgroups go to the 8 XCDs in turn; XCD_RUN neighbouring heads (whose rows of a step lie
// together) go to one of them, so that what one L2 fetches lies together too. (256 steps of 2,000 envs, 8 heads of 32, bf16: 337 us,
// 481 with one; 128 steps of 2,056 envs, 8 heads of 64: 282 and 292.)
constexpr int XCD_RUN = 16;
__device__ __forceinline__ int64_t head_of_block(int64_t heads) {
    const int64_t b = block_here(), round = 8 * XCD_RUN;
    if (b >= heads / round * round) return b;
    return b / round * round + b % 8 * XCD_RUN + b % round / 8;
}

// A long sequence is cut into segments of whole chunks, a workgroup each, so that few sequences fill the chip. First each
// segment's own sum and what it leaves of an entering state (`keep`: g^steps, or -1 where an episode starts inside), then the
// states that enter the segments one after another, then the outputs from there. (16,001 steps of 2 envs with 8 heads of 128, bf16: 48
// us for the sums, 15 for the states between, 102 for the outputs under the profiler, 144 in all without; k and v are read twice.)
struct Cut {
    int64_t chunks, per_seg;   // chunks of a sequence and of a segment
    int segs;
    float* enter;              // (segs, N H, D E): a segment's own sum, then the state that enters it
    float* keep;               // (segs, N H)
};

enum { KEEP_NONE = 0, KEEP_STATES = 1, ONLY_SUMS = 2 };

// MODE: KEEP_STATES leaves the states that enter chunks 1, 2, .. for the gradient in a.saved, (N H, chunks - 1, P, P) in float32.
// ONLY_SUMS makes a segment's own sum.
// A wave's 16 columns (from x0) of a head's float32 (D, E) matrix, or of its transpose, to and from accumulator tiles. Of the
// transpose a lane has four neighbours, moved together (E is a multiple of 4).
struct alignas(4) Four { float v[4]; };
template <int P, bool TRANSPOSED, class F> __device__ __forceinline__ void each_of_state(const MoAttend& a, int x0, F f) {
    const int lane = threadIdx.x % kWave, g = lane / 16, x = x0 + lane % 16;
    const auto tiles = [&](auto whole) {                       // (whole heads without a test and with known strides)
        const int E = whole ? P : a.E;
#pragma unroll
        for (int t = 0; t < P / 16; t++) {
            const int y = acc_row(t, g, 0);
            if (TRANSPOSED) {
                if (whole || (x < a.D && y < a.E)) f(t, 0, x * E + y);
            } else {
#pragma unroll
                for (int r = 0; r < 4; r++)
                    if (whole || (y + r < a.D && x < a.E)) f(t, r, (y + r) * E + x);
            }
        }
    };
    if (!TRANSPOSED && a.D == P && a.E == P) tiles(std::true_type{});
    else tiles(std::false_type{});
}
template <int P, bool TRANSPOSED> __device__ __forceinline__ void load_state(const MoAttend& a, const float* from, int x0, f32x4 (&S)[P / 16]) {
    each_of_state<P, TRANSPOSED>(a, x0, [&](int t, int r, int at) {
        if (!TRANSPOSED) { S[t][r] = from[at]; return; }
        const Four q = *(const Four*)(from + at);
#pragma unroll
        for (int i = 0; i < 4; i++) S[t][i] = q.v[i];
    });
}
template <int P, bool TRANSPOSED> __device__ __forceinline__ void store_state(const MoAttend& a, float* to, int x0, const f32x4 (&S)[P / 16]) {
    each_of_state<P, TRANSPOSED>(a, x0, [&](int t, int r, int at) {
        if (!TRANSPOSED) to[at] = S[t][r];
        else *(Four*)(to + at) = Four{{S[t][0], S[t][1], S[t][2], S[t][3]}};
    });
}

// Where a step does not see another, their product's factor is 0; but 0 times a NaN or an infinity is a NaN, which would reach
// steps of other episodes. Such a value shows in every sum that it entered, so sums that are not finite are made again over
// what is seen only, one product after another. (`all` adds the sums up: it is not finite if one of them is not.)
__device__ __forceinline__ void watch(float& all, const f32x4& x) { all += (x[0] + x[1]) + (x[2] + x[3]); }
__device__ __forceinline__ bool any_not_finite(float all) { return __ballot(!(fabsf(all) < INFINITY)) != 0; }

template <int P> constexpr int kForwardWaves = P / 16 < 4 ? P / 16 : 4;
template <int P> constexpr int kForwardPerSimd = P == 128 ? 2 : 3;   // waves a SIMD: what LDS leaves room for

template <class T, int P, int MODE>
__global__ void __launch_bounds__((kForwardWaves<P> * kWave), (kForwardPerSimd<P>)) k_attend(MoAttend a, Cut cut) {
    typedef Chunk<T, P, kForwardWaves<P>> C;
    typedef HeadRows<T, C> Head;
    constexpr int L = C::L, CT = C::CT, K = C::K;
    constexpr bool OUT = MODE != ONLY_SUMS;
    __shared__ __align__(16) T lk[L * P], lv[L * P], lq[OUT ? L * P : 8], lp[OUT ? C::SCORES : 8], ly[OUT ? L * P : 8];
    __shared__ Powers<L> pw;
    __shared__ __align__(16) float wt[L];
    __shared__ float rt[OUT ? L : 1];   // what a step has of the entering state: scale g^(i+1), or 0
    const typename C::Rows sk{lk}, sv{lv}, sq{lq}, sy{ly};
    const typename C::Scored sp(lp);
    const int w = threadIdx.x / kWave;
    const int64_t nh = head_of_block(a.N * a.H), env = nh / a.H;
    if (nh >= a.N * a.H) return;
    const int h = (int)(nh % a.H), seg = blockIdx.y;
    const int64_t c0 = seg * cut.per_seg, c1 = min(c0 + cut.per_seg, cut.chunks);
    const int e0 = w * CT * 16;   // the wave's columns
    const int64_t de = (int64_t)a.D * a.E;
    const Head k(a.k, env, h, a.D, a.D == P), v(a.v, env, h, a.E, a.E == P), q(a.q, env, h, a.D, a.D == P), out(a.out, env, h, a.E, on_pieces<T>(a.out));
    const f32x4 zero = {0.f, 0.f, 0.f, 0.f};

    f32x4 S[CT][C::PT];
#pragma unroll
    for (int ct = 0; ct < CT; ct++)
#pragma unroll
        for (int dt = 0; dt < C::PT; dt++) S[ct][dt] = zero;
    const float* in = !OUT ? nullptr : cut.segs > 1 ? cut.enter + ((int64_t)seg * a.N * a.H + nh) * de : a.state ? a.state + nh * de : nullptr;
    if (in)
#pragma unroll
        for (int ct = 0; ct < CT; ct++) load_state<P, false>(a, in, e0 + 16 * ct, S[ct]);
    pw.fill(a.decay[h], a.scale);
    bool any_start = false;
    for (int64_t c = c0; c < c1; c++) {
        const int64_t t0 = c * L;
        const int n = (int)min((int64_t)L, a.T - t0);
        __syncthreads();                                       // the last chunk's tiles are done with, its outputs in theirs
        k.bring(lk, t0, n);
        v.bring(lv, t0, n);
        if (OUT) q.bring(lq, t0, n);
        if (OUT && c > c0) out.take(ly, t0 - L, L);
        const uint64_t m = __ballot(start_of_lane(a, t0, n, env) != 0);   // the chunk's starts as bits
        any_start |= m != 0;
        const int last = seen_from(m, L - 1);
        if (threadIdx.x < L) {
            const int i = threadIdx.x;
            wt[i] = i < n && i >= last ? pw.pw[n - 1 - i] : 0.f;
            if (OUT) rt[i] = seen_from(m, i) < 0 ? a.scale * pw.pw[i + 1] : 0.f;
        }
        brought();
        const unsigned lane = thread_here() % kWave, g = lane / 16, i16 = lane % 16;

        if (OUT) {
            // scores, transposed: a lane has four neighbouring j of one i
            const auto scores = [&](auto starts) {
#pragma unroll
                for (int x = 0; x < C::TPW; x++) {
                    const int idx = w + x * C::WAVES;
                    if (C::TILES % C::WAVES && idx >= C::TILES) break;
                    int it, jt;
                    C::score_tile(idx, it, jt);
                    f32x4 s = zero;
#pragma unroll
                    for (int b = 0; b < C::PB; b++) mma(s, sk.along(jt * 16, b * 32, lane), sq.along(it * 16, b * 32, lane));
                    const int i = it * 16 + i16, j = jt * 16 + 4 * g, from = starts ? seen_from(m, i) : 0;
                    const float* f = pw.sees(i, j);
#pragma unroll
                    for (int r = 0; r < 4; r++) s[r] = !starts || j + r >= from ? s[r] * f[-r] : 0.f;
                    sp.put(i, j, s);
                }
            };
            if (m) scores(std::true_type{});
            else scores(std::false_type{});
            if (MODE == KEEP_STATES && c > 0) {                // (copied as they lie: what is not finite stays in its row and column)
                float* to = (float*)a.saved + (nh * (cut.chunks - 1) + c - 1) * (P * P) + e0 + i16;
#pragma unroll
                for (int ct = 0; ct < CT; ct++)
#pragma unroll
                    for (int t = 0; t < C::PT; t++)
#pragma unroll
                        for (int r = 0; r < 4; r++) to[acc_row(t, g, r) * P + ct * 16] = S[ct][t][r];
            }
            __syncthreads();
        }

        Frag<T> vf[CT][C::LB];
#pragma unroll
        for (int ct = 0; ct < CT; ct++)
#pragma unroll
            for (int b = 0; b < C::LB; b++) vf[ct][b] = sv.down(b * 32, e0 + 16 * ct, lane);

        if (OUT) {
            // outputs, transposed: a lane has four neighbouring columns of one step
            const auto write = [&](int it, int ct, const f32x4& own, const f32x4& far) {
                const float f = rt[it * 16 + i16];
                f32x4 x;
#pragma unroll
                for (int r = 0; r < 4; r++) x[r] = fmaf(f, far[r], own[r]);
                if (m && f == 0.f) x = own;                    // (a state that is not seen may be anything)
                *(Pack<T, 4>*)sy.at(it * 16 + i16, e0 + 16 * ct + 4 * g) = pack4(x, T{});
            };
            float all = 0.f;
            {
                Frag<T> sf[CT][C::PB][K];
#pragma unroll
                for (int ct = 0; ct < CT; ct++)
#pragma unroll
                    for (int b = 0; b < C::PB; b++) halves<T>(S[ct][2 * b], S[ct][2 * b + 1], sf[ct][b]);
#pragma unroll
                for (int it = 0; it < C::LT; it++) {
                    f32x4 own[CT], far[CT];
#pragma unroll
                    for (int ct = 0; ct < CT; ct++) { own[ct] = zero; far[ct] = zero; }
#pragma unroll
                    for (int b = 0; b < C::PB; b++) {
                        const Frag<T> x = sq.along(it * 16, b * 32, lane);
#pragma unroll
                        for (int p = 0; p < K; p++)
#pragma unroll
                            for (int ct = 0; ct < CT; ct++) mma(far[ct], sf[ct][b][p], x);
                    }
#pragma unroll
                    for (int b = 0; b <= it / 2; b++)
#pragma unroll
                        for (int p = 0; p < K; p++) {
                            const Frag<T> x = sp.part[p].along(it * 16, b * 32, lane);
#pragma unroll
                            for (int ct = 0; ct < CT; ct++) mma(own[ct], vf[ct][b], x);
                        }
#pragma unroll
                    for (int ct = 0; ct < CT; ct++) {
                        watch(all, own[ct]);
                        write(it, ct, own[ct], far[ct]);
                    }
                }
            }
            if (any_not_finite(all)) {
#pragma unroll
                for (int ct = 0; ct < CT; ct++)
#pragma unroll 1
                    for (int it = 0; it < C::LT; it++) {
                        const int i = it * 16 + i16;
                        f32x4 own = zero, far = zero;
#pragma unroll
                        for (int b = 0; b < C::PB; b++) {
                            Frag<T> sf[K];
                            halves<T>(S[ct][2 * b], S[ct][2 * b + 1], sf);
                            const Frag<T> x = sq.along(it * 16, b * 32, lane);
#pragma unroll
                            for (int p = 0; p < K; p++) mma(far, sf[p], x);
                        }
#pragma unroll 1
                        for (int j = max(seen_from(m, i), 0); j <= i; j++)
#pragma unroll
                            for (int r = 0; r < 4; r++)
                                own[r] = fmaf(sp.get(i, j), as_f32(*sv.at(j, e0 + 16 * ct + 4 * g + r)), own[r]);
                        write(it, ct, own, far);
                    }
            }
        }

        f32x4 add[CT][C::PT];
#pragma unroll
        for (int ct = 0; ct < CT; ct++)
#pragma unroll
            for (int dt = 0; dt < C::PT; dt++) add[ct][dt] = zero;
#pragma unroll
        for (int b = 0; b < C::LB; b++) {
            Frag<T> part[CT][kParts<T>];
#pragma unroll
            for (int ct = 0; ct < CT; ct++) scaled_parts(vf[ct][b], &wt[b * 32 + 8 * g], part[ct]);
#pragma unroll
            for (int dt = 0; dt < C::PT; dt++) {
                const Frag<T> kf = sk.template down<true>(b * 32, acc_col(dt), lane);
#pragma unroll
                for (int p = 0; p < kParts<T>; p++)
#pragma unroll
                    for (int ct = 0; ct < CT; ct++) mma(add[ct][dt], kf, part[ct][p]);
            }
        }
        float all = 0.f;
#pragma unroll
        for (int ct = 0; ct < CT; ct++)
#pragma unroll
            for (int dt = 0; dt < C::PT; dt++) watch(all, add[ct][dt]);
        if (any_not_finite(all)) {
#pragma unroll
            for (int ct = 0; ct < CT; ct++)
#pragma unroll
                for (int dt = 0; dt < C::PT; dt++) {
                    add[ct][dt] = zero;
#pragma unroll 1
                    for (int j = max(last, 0); j < n; j++)
#pragma unroll
                        for (int r = 0; r < 4; r++)
                            add[ct][dt][r] = fmaf(wt[j] * as_f32(*sk.at(j, acc_row(dt, g, r))), as_f32(*sv.at(j, e0 + 16 * ct + i16)), add[ct][dt][r]);
                }
        }
        const float f = pw.pw[n];
#pragma unroll
        for (int ct = 0; ct < CT; ct++)
#pragma unroll
            for (int dt = 0; dt < C::PT; dt++)
#pragma unroll
                for (int r = 0; r < 4; r++) S[ct][dt][r] = last < 0 ? fmaf(f, S[ct][dt][r], add[ct][dt][r]) : add[ct][dt][r];
    }
    if (OUT && c0 < c1) {
        __syncthreads();
        out.take(ly, (c1 - 1) * L, (int)min((int64_t)L, a.T - (c1 - 1) * L));
    }
    float* to = !OUT ? cut.enter + ((int64_t)seg * a.N * a.H + nh) * de : cut.segs > 1 ? nullptr : a.state_out + nh * de;
    if (to)
#pragma unroll
        for (int ct = 0; ct < CT; ct++) store_state<P, false>(a, to, e0 + 16 * ct, S[ct]);
    if (!OUT && threadIdx.x == 0) {
        const int64_t n = min(c1 * L, a.T) - c0 * L;
        cut.keep[(int64_t)seg * a.N * a.H + nh] = any_start ? -1.f : power(a.decay[h], n);
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
// The chunk kernels take heads of whole 16-byte pieces whose rows lie on them; the rest goes step by step (k_walk; 128 steps of
// 1,000 envs, 8 heads, bf16: heads of 40 by chunks 214 us, with the gradient 646; heads of 36 step by step 854 and 3,370).
inline bool chunks_take(const MoAttend& a, bool backward) {
    const int64_t epv = a.dtype == MO_BF16 ? 8 : 4;
    if (a.T == 0 || a.D % epv || a.E % epv || !rows_suit(a.q, epv) || !rows_suit(a.k, epv) || !rows_suit(a.v, epv)) return false;
    return !backward || rows_suit(a.dout, epv);
}
inline int chunk_steps(const MoAttend& a) { return a.dtype == MO_BF16 ? 64 : 32; }
inline int padded_head(const MoAttend& a) { const int m = std::max(a.D, a.E); return m <= 32 ? 32 : m <= 64 ? 64 : 128; }

// Segments: up to two workgroups a compute unit, of two chunks at least. Two segments are not worth it: k, v (or q, dO) are read
// twice and two more kernels run. (16,001 steps of 16 heads of 128: 1,560 us in one piece, 159 in 32; 2,000 steps of 512 heads of
// 64: 145 in one piece, 210 in two; 300 steps of 32 heads of 128: 35 in one, 41 in two.)
inline Cut attend_cut(const MoAttend& a) {
    Cut c{};
    c.chunks = (a.T + chunk_steps(a) - 1) / chunk_steps(a);
    const int64_t segs = std::min<int64_t>(2 * (int64_t)compute_units() / std::max<int64_t>(1, a.N * a.H), c.chunks / 2);
    c.per_seg = segs < 3 ? std::max<int64_t>(1, c.chunks) : (c.chunks + segs - 1) / segs;
    c.segs = (int)std::max<int64_t>(1, (c.chunks + c.per_seg - 1) / c.per_seg);
    return c;
}
inline int64_t saved_bytes(const MoAttend& a) {
    const int64_t p = padded_head(a);
    return a.N * a.H * ((a.T + chunk_steps(a) - 1) / chunk_steps(a) - 1) * p * p * 4;
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

template <class T, int P> int attend_chunks(const MoAttend& a, hipStream_t s) {
    Cut c = attend_cut(a);
    cut_place(a, c);
    const dim3 grid = grid_of(a.N * a.H, c.segs), block(kForwardWaves<P> * kWave);
    if (c.segs > 1) {
        hipLaunchKernelGGL((k_attend<T, P, ONLY_SUMS>), grid, block, 0, s, a, c);
        if (launched("k_attend sums") || enter_states(a, c, a.state, a.state_out, false, s)) return -1;
    }
    if (a.saved && c.chunks > 1) hipLaunchKernelGGL((k_attend<T, P, KEEP_STATES>), grid, block, 0, s, a, c);
    else hipLaunchKernelGGL((k_attend<T, P, KEEP_NONE>), grid, block, 0, s, a, c);
    return launched("k_attend");
}

}  // namespace mo
