// Linear attention by chunks of steps on the matrix cores: the gradient.
#pragma once
#include "attend_chunk.hpp"

namespace mo {

// Backwards over the chunks, with R the gradient of the state that leaves a chunk, S the state that enters it, and G and w as
// in the forward pass. With A = scale Q K^T . G and B = scale dO V^T . G (both L x L):
//   dQ = B K + scale diag(g^(i+1), 0 past the first start) dO S^T
//   dK = B^T Q + diag(w) V R^T
//   dV = A^T dO + diag(w) K R
//   R' = (no start in the chunk ? g^n : 0) R + Q^T diag(u) dO,   u_i = scale g^(i+1), 0 past the first start
// q, k, v and dO are read once for all of them. Wave w holds the 16 rows of R from 16 w, as the accumulator tiles of R^T, which
// are the operand of V R^T as they lie; K R takes R from LDS. S comes from the forward pass (a.saved), each wave its rows, in
// 16-byte pieces straight into operands.
template <class T, int P> struct BackLds {
    typedef Chunk<T, P> C;
    T q[C::L][C::LD], k[C::L][C::LD], v[C::L][C::LD], o[C::L][C::LD];   // o: dO
    T a[C::L][C::LS], b[C::L][C::LS];
    T r[P][C::LD];
    float pw[C::L + 4], wt[C::L], ut[C::L];
    int odd[4];
};

template <class T, int P>
__global__ void __launch_bounds__((Chunk<T, P>::NT)) k_attend_back(MoAttend a, Cut cut) {
    typedef Chunk<T, P> C;
    constexpr int L = C::L;
    extern __shared__ __align__(16) char lds[];
    BackLds<T, P>& s = *(BackLds<T, P>*)lds;
    const int lane = threadIdx.x % kWave, w = threadIdx.x / kWave, g = lane / 16, i16 = lane % 16;
    const int64_t nh = blockIdx.x, env = nh / a.H;
    const int h = (int)(nh % a.H), seg = blockIdx.y;
    const int64_t c0 = seg * cut.per_seg, c1 = min(c0 + cut.per_seg, cut.chunks);
    const int x0 = w * 16;     // the wave's rows of R and S, columns of dq and dk; of dv its columns
    const int64_t de = (int64_t)a.D * a.E;

    powers<L>(s.pw, a.decay[h]);
    if (threadIdx.x < 2) s.odd[threadIdx.x] = 0;
    f32x4 R[C::PT];            // R^T: rows e, columns d
    const float* in = cut.segs > 1 ? cut.enter + ((int64_t)seg * a.N * a.H + nh) * de : a.dstate_out ? a.dstate_out + nh * de : nullptr;
#pragma unroll
    for (int et = 0; et < C::PT; et++)
#pragma unroll
        for (int r = 0; r < 4; r++) {
            const int d = x0 + i16, e = et * 16 + 4 * g + r;
            R[et][r] = in && d < a.D && e < a.E ? in[d * a.E + e] : 0.f;
        }
    Rows<T, P> q, k, v, o;
    q.init(a.q, env, h, a.D);
    k.init(a.k, env, h, a.D);
    v.init(a.v, env, h, a.E);
    o.init(a.dout, env, h, a.E);
    const auto steps = [&](int64_t c) { return (int)min((int64_t)L, a.T - c * L); };
    int starts = 0;
    const auto fetch = [&](int64_t c) {
        const int n = steps(c);
        starts = start_of_lane(a, c * L, n, env);
        q.load(c * L, n);
        k.load(c * L, n);
        v.load(c * L, n);
        o.load(c * L, n);
    };
    if (c0 < c1) fetch(c1 - 1);
    for (int64_t c = c1 - 1; c >= c0; c--) {
        const int n = steps(c);
        const int64_t t0 = c * L;
        __syncthreads();                                       // the last chunk's tiles are done with
        q.put(s.q);
        k.put(s.k);
        v.put(s.v);
        o.put(s.o);
#pragma unroll
        for (int et = 0; et < C::PT; et++) {
            Pack<T, 4> x;
#pragma unroll
            for (int r = 0; r < 4; r++) x.v[r] = as<T>(R[et][r]);
            *(Pack<T, 4>*)&s.r[x0 + i16][et * 16 + 4 * g] = x;
        }
        const uint64_t m = __ballot(starts != 0);
        const int last = seen_from(m, L - 1);
        if (threadIdx.x < L) {
            const int i = threadIdx.x;
            s.wt[i] = i < n && i >= last ? s.pw[n - 1 - i] : 0.f;
            s.ut[i] = i < n && seen_from(m, i) < 0 ? a.scale * s.pw[i + 1] : 0.f;
        }
        if (not_finite(q.most(k.most(v.most(o.most(0)))), T{})) s.odd[c & 1] = 1;
        __syncthreads();
        if (c > c0) fetch(c - 1);
        const bool exact_sums = s.odd[c & 1];
        if (threadIdx.x == 0) s.odd[(c + 1) & 1] = 0;
        // the state that enters the chunk: rows d of the wave, eight neighbouring columns e a lane
        Frag<T> sf[C::PB];
        {
            const int d = x0 + i16;
            const T* kept = c > 0 && a.saved ? (const T*)a.saved + (nh * (cut.chunks - 1) + c - 1) * de : nullptr;
#pragma unroll
            for (int b = 0; b < C::PB; b++) {
                const int e = b * 32 + 8 * g;
                const bool in = d < a.D && e < a.E;
                if (c > 0) {
                    union { uint4 u[sizeof(T) / 2]; T x[8]; } y{};
                    if (in)
#pragma unroll
                        for (int j = 0; j < (int)sizeof(T) / 2; j++)
                            if (e + j * C::EPV < a.E) y.u[j] = *(const uint4*)(kept + d * a.E + e + j * C::EPV);
#pragma unroll
                    for (int j = 0; j < 8; j++) sf[b].v[j] = y.x[j];
                } else {
#pragma unroll
                    for (int j = 0; j < 8; j++)
                        sf[b].v[j] = as<T>(a.state && in && e + j < a.E ? a.state[nh * de + d * a.E + e + j] : 0.f);
                }
            }
        }

        for (int idx = w; idx < C::TILES; idx += C::WAVES) {   // A and B, a lane four neighbouring j of one i
            int it, jt;
            C::score_tile(idx, it, jt);
            f32x4 x = {0.f, 0.f, 0.f, 0.f}, y = {0.f, 0.f, 0.f, 0.f};
            if (jt <= it) {
#pragma unroll
                for (int b = 0; b < C::PB; b++) {
                    mma(x, frag_in_order(&s.k[jt * 16 + i16][b * 32], g), frag_in_order(&s.q[it * 16 + i16][b * 32], g));
                    mma(y, frag_in_order(&s.v[jt * 16 + i16][b * 32], g), frag_in_order(&s.o[it * 16 + i16][b * 32], g));
                }
                const int i = it * 16 + i16, j = jt * 16 + 4 * g, from = seen_from(m, i);
#pragma unroll
                for (int r = 0; r < 4; r++) {
                    const bool sees = j + r <= i && j + r >= from;
                    const float f = a.scale * s.pw[max(i - j - r, 0)];
                    x[r] = sees ? f * x[r] : 0.f;
                    y[r] = sees ? f * y[r] : 0.f;
                }
            }
            Pack<T, 4> xa, yb;
#pragma unroll
            for (int r = 0; r < 4; r++) { xa.v[r] = as<T>(x[r]); yb.v[r] = as<T>(y[r]); }
            *(Pack<T, 4>*)&s.a[it * 16 + i16][jt * 16 + 4 * g] = xa;
            *(Pack<T, 4>*)&s.b[it * 16 + i16][jt * 16 + 4 * g] = yb;
        }
        __syncthreads();

        // Each output transposed: a lane has four neighbouring columns of one step. `own` the sum over the chunk's steps, `far`
        // what the entering state or its gradient adds, by a factor a step.
        f32x4 own[C::LT], far[C::LT];
        const auto clear = [&] {
#pragma unroll
            for (int t = 0; t < C::LT; t++) { own[t] = f32x4{0.f, 0.f, 0.f, 0.f}; far[t] = own[t]; }
        };
        const auto write = [&](const MoRows& to, int size, auto factor) {
            const bool wide = rows_wide(to, 4 * sizeof(T));
            T* p = (T*)to.p + env * to.sn + h * to.sh + x0 + 4 * g;
            if (x0 + 4 * g >= size) return;
#pragma unroll
            for (int t = 0; t < C::LT; t++) {
                const int i = t * 16 + i16;
                if (i >= n) continue;
                const float f = factor(i);
                Pack<T, 4> y;
#pragma unroll
                for (int r = 0; r < 4; r++) y.v[r] = as<T>(f == 0.f ? own[t][r] : fmaf(f, far[t][r], own[t][r]));
                put4(p + (t0 + i) * to.st, y, wide);
            }
        };

        clear();                                               // dQ
        if (!exact_sums) {
            Frag<T> kf[C::LB];
#pragma unroll
            for (int b = 0; b < C::LB; b++) kf[b] = frag_down(&s.k[b * 32][x0], C::LD, lane);
#pragma unroll
            for (int t = 0; t < C::LT; t++)
#pragma unroll
                for (int b = 0; b <= t / 2; b++) mma(own[t], kf[b], frag_in_order(&s.b[t * 16 + i16][b * 32], g));
        } else {
#pragma unroll
            for (int t = 0; t < C::LT; t++) {
                const int i = t * 16 + i16;
                for (int j = max(seen_from(m, i), 0); j <= i; j++)
#pragma unroll
                    for (int r = 0; r < 4; r++) own[t][r] = fmaf(as_f32(s.b[i][j]), as_f32(s.k[j][x0 + 4 * g + r]), own[t][r]);
            }
        }
#pragma unroll
        for (int b = 0; b < C::PB; b++)
#pragma unroll
            for (int t = 0; t < C::LT; t++) mma(far[t], sf[b], frag_in_order(&s.o[t * 16 + i16][b * 32], g));
        write(a.dq, a.D, [&](int i) { return s.ut[i]; });

        clear();                                               // dK
        Frag<T> qf[C::LB], of[C::LB];
#pragma unroll
        for (int b = 0; b < C::LB; b++) qf[b] = frag_down(&s.q[b * 32][x0], C::LD, lane);
        if (!exact_sums) {
#pragma unroll
            for (int t = 0; t < C::LT; t++)
#pragma unroll
                for (int b = t / 2; b < C::LB; b++) mma(own[t], qf[b], frag_down(&s.b[b * 32][t * 16], C::LS, lane));
        } else {
#pragma unroll
            for (int t = 0; t < C::LT; t++) {
                const int j = t * 16 + i16;
                for (int i = j; i < n && seen_from(m, i) <= j; i++)
#pragma unroll
                    for (int r = 0; r < 4; r++) own[t][r] = fmaf(as_f32(s.b[i][j]), as_f32(s.q[i][x0 + 4 * g + r]), own[t][r]);
            }
        }
#pragma unroll
        for (int b = 0; b < C::PB; b++) {
            const Frag<T> rf = state_frag<T>(R[2 * b], R[2 * b + 1]);
#pragma unroll
            for (int t = 0; t < C::LT; t++) mma(far[t], rf, frag_in_halves(&s.v[t * 16 + i16][b * 32], g));
        }
        write(a.dk, a.D, [&](int i) { return s.wt[i]; });

        clear();                                               // dV
        if (!exact_sums) {
#pragma unroll
            for (int b = 0; b < C::LB; b++) of[b] = frag_down(&s.o[b * 32][x0], C::LD, lane);
#pragma unroll
            for (int t = 0; t < C::LT; t++)
#pragma unroll
                for (int b = t / 2; b < C::LB; b++) mma(own[t], of[b], frag_down(&s.a[b * 32][t * 16], C::LS, lane));
        } else {
#pragma unroll
            for (int t = 0; t < C::LT; t++) {
                const int j = t * 16 + i16;
                for (int i = j; i < n && seen_from(m, i) <= j; i++)
#pragma unroll
                    for (int r = 0; r < 4; r++) own[t][r] = fmaf(as_f32(s.a[i][j]), as_f32(s.o[i][x0 + 4 * g + r]), own[t][r]);
            }
        }
#pragma unroll
        for (int b = 0; b < C::PB; b++) {
            const Frag<T> rf = frag_down(&s.r[b * 32][x0], C::LD, lane);
#pragma unroll
            for (int t = 0; t < C::LT; t++) mma(far[t], rf, frag_in_order(&s.k[t * 16 + i16][b * 32], g));
        }
        write(a.dv, a.E, [&](int i) { return s.wt[i]; });

        const float f = s.pw[n];                               // R'
        if (!exact_sums) {
            Frag<T> part[C::LB][kParts<T>];
#pragma unroll
            for (int b = 0; b < C::LB; b++) scaled_parts(qf[b], &s.ut[b * 32 + 8 * g], part[b]);
#pragma unroll
            for (int et = 0; et < C::PT; et++) {
#pragma unroll
                for (int r = 0; r < 4; r++) R[et][r] = m ? 0.f : f * R[et][r];
#pragma unroll
                for (int b = 0; b < C::LB; b++) {
                    const Frag<T> x = frag_down(&s.o[b * 32][et * 16], C::LD, lane);
#pragma unroll
                    for (int p = 0; p < kParts<T>; p++) mma(R[et], x, part[b][p]);
                }
            }
        } else {
            const int first = m ? (int)__ffsll((long long)m) - 1 : n;
#pragma unroll
            for (int et = 0; et < C::PT; et++)
#pragma unroll
                for (int r = 0; r < 4; r++) {
                    float x = m ? 0.f : f * R[et][r];
                    for (int i = 0; i < first; i++) x = fmaf(s.ut[i] * as_f32(s.q[i][x0 + i16]), as_f32(s.o[i][et * 16 + 4 * g + r]), x);
                    R[et][r] = x;
                }
        }
    }
    if (!a.dstate || cut.segs > 1) return;
#pragma unroll
    for (int et = 0; et < C::PT; et++)
#pragma unroll
        for (int r = 0; r < 4; r++) {
            const int d = x0 + i16, e = et * 16 + 4 * g + r;
            if (d < a.D && e < a.E) a.dstate[nh * de + d * a.E + e] = R[et][r];
        }
}

// A segment's own sum of R' (see R' above) and what it leaves of a gradient that comes from behind it.
template <class T, int P>
__global__ void __launch_bounds__((Chunk<T, P>::NT)) k_attend_back_sums(MoAttend a, Cut cut) {
    typedef Chunk<T, P> C;
    constexpr int L = C::L;
    __shared__ __align__(16) T sq[L][C::LD], so[L][C::LD];
    __shared__ float pw[L + 1];
    __shared__ __align__(16) float ut[L];
    __shared__ int odd[2];
    const int lane = threadIdx.x % kWave, w = threadIdx.x / kWave, g = lane / 16, i16 = lane % 16;
    const int64_t nh = blockIdx.x, env = nh / a.H;
    const int h = (int)(nh % a.H), seg = blockIdx.y;
    const int64_t c0 = seg * cut.per_seg, c1 = min(c0 + cut.per_seg, cut.chunks);
    const int x0 = w * 16;
    powers<L>(pw, a.decay[h]);
    if (threadIdx.x < 2) odd[threadIdx.x] = 0;
    f32x4 R[C::PT];
#pragma unroll
    for (int et = 0; et < C::PT; et++) R[et] = f32x4{0.f, 0.f, 0.f, 0.f};
    Rows<T, P> q, o;
    q.init(a.q, env, h, a.D);
    o.init(a.dout, env, h, a.E);
    const auto steps = [&](int64_t c) { return (int)min((int64_t)L, a.T - c * L); };
    int starts = 0;
    const auto fetch = [&](int64_t c) {
        starts = start_of_lane(a, c * L, steps(c), env);
        q.load(c * L, steps(c));
        o.load(c * L, steps(c));
    };
    if (c0 < c1) fetch(c1 - 1);
    bool any_start = false;
    for (int64_t c = c1 - 1; c >= c0; c--) {
        const int n = steps(c);
        __syncthreads();
        q.put(sq);
        o.put(so);
        const uint64_t m = __ballot(starts != 0);
        any_start |= m != 0;
        if (threadIdx.x < L) ut[threadIdx.x] = (int)threadIdx.x < n && seen_from(m, threadIdx.x) < 0 ? a.scale * pw[threadIdx.x + 1] : 0.f;
        if (not_finite(q.most(o.most(0)), T{})) odd[c & 1] = 1;
        __syncthreads();
        if (c > c0) fetch(c - 1);
        const bool exact_sums = odd[c & 1];
        if (threadIdx.x == 0) odd[(c + 1) & 1] = 0;
        const float f = pw[n];
        if (!exact_sums) {
            Frag<T> part[C::LB][kParts<T>];
#pragma unroll
            for (int b = 0; b < C::LB; b++) scaled_parts(frag_down(&sq[b * 32][x0], C::LD, lane), &ut[b * 32 + 8 * g], part[b]);
#pragma unroll
            for (int et = 0; et < C::PT; et++) {
#pragma unroll
                for (int r = 0; r < 4; r++) R[et][r] = m ? 0.f : f * R[et][r];
#pragma unroll
                for (int b = 0; b < C::LB; b++) {
                    const Frag<T> x = frag_down(&so[b * 32][et * 16], C::LD, lane);
#pragma unroll
                    for (int p = 0; p < kParts<T>; p++) mma(R[et], x, part[b][p]);
                }
            }
        } else {
            const int first = m ? (int)__ffsll((long long)m) - 1 : n;
#pragma unroll
            for (int et = 0; et < C::PT; et++)
#pragma unroll
                for (int r = 0; r < 4; r++) {
                    float x = m ? 0.f : f * R[et][r];
                    for (int i = 0; i < first; i++) x = fmaf(ut[i] * as_f32(sq[i][x0 + i16]), as_f32(so[i][et * 16 + 4 * g + r]), x);
                    R[et][r] = x;
                }
        }
    }
    float* to = cut.enter + ((int64_t)seg * a.N * a.H + nh) * a.D * a.E;
#pragma unroll
    for (int et = 0; et < C::PT; et++)
#pragma unroll
        for (int r = 0; r < 4; r++) {
            const int d = x0 + i16, e = et * 16 + 4 * g + r;
            if (d < a.D && e < a.E) to[d * a.E + e] = R[et][r];
        }
    if (threadIdx.x == 0) {
        const int64_t n = min(c1 * L, a.T) - c0 * L;
        cut.keep[(int64_t)seg * a.N * a.H + nh] = any_start ? -1.f : exp2f((float)n * __log2f(a.decay[h]));
    }
}

constexpr int BACKWARD_PER_CU = 2;

template <class T, int P> int attend_back_chunks(const MoAttend& a, hipStream_t s) {
    Cut c = attend_cut(a, BACKWARD_PER_CU);
    cut_place(a, c);
    const dim3 grid((unsigned)(a.N * a.H), (unsigned)c.segs), block(Chunk<T, P>::NT);
    if (c.segs > 1) {
        hipLaunchKernelGGL((k_attend_back_sums<T, P>), grid, block, 0, s, a, c);
        if (launched("k_attend_back_sums") || enter_states(a, c, a.dstate_out, a.dstate, true, s)) return -1;
    }
    hipLaunchKernelGGL((k_attend_back<T, P>), grid, block, sizeof(BackLds<T, P>), s, a, c);
    return launched("k_attend_back");
}

}  // namespace mo
