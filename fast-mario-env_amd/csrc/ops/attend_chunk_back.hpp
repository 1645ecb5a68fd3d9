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
// 16-byte pieces. A, B, R and S go into products in two parts each (halves, in tiles.hpp); to leave LDS room for two workgroups of heads of
// 64 a compute unit, B waits in registers until A is done with, and dV until R is.
//
// 4 rows are read and 3 written a step and head, and a state a chunk. Measured, bf16, from zeros, the gradient of 128 steps of 2,056 envs with 8
// heads of 64: 596 us, 3.6 TB/s (500 with one part of A, B, R and S; 730 at 2,048 envs, whose steps' rows lie a multiple of 2 MiB apart):
// neither memory nor the matrix units (13 % busy) are full, waves wait 43 % of their time with two workgroups a compute unit. Heads of 128,
// 1,000 envs: 916 us, 2.6 TB/s (702): the tiles leave room for one workgroup a compute unit, whose loads wait while it multiplies, and 256
// registers spill 12. float32 holds half the steps in as much LDS and its matrix instructions take 16 times as long: the 1,000 envs with heads
// of 64 take 672 us, in bf16 291; at 97 steps of 64 envs its matrix units are busy 51 % of the time. Step by step (k_walk, three walks): 128
// steps of 2,048 envs with the forward pass 10,277 us, 1,312 by chunks.
template <class T, int P> using BackChunk = Chunk<T, P, P / 16>;
template <class T, int P> struct BackLds {
    typedef BackChunk<T, P> C;
    static constexpr int L = C::L, ROWS = L * P;
    T q[ROWS], k[ROWS], v[ROWS], o[ROWS];        // o: dO
    T x[C::SCORES];                              // A, then B
    T r[C::K * P * P > 3 * ROWS ? C::K * P * P : 3 * ROWS];
    float wt[L], ut[L];
    Powers<L> pw;
    // Once dV is made, R's tiles have room for the results.
    __device__ __forceinline__ T* dv() { return r; }
    __device__ __forceinline__ T* dq() { return r + ROWS; }
    __device__ __forceinline__ T* dk() { return r + 2 * ROWS; }
};

// The sum over a chunk's steps of Q^T diag(u) dO, as R^T's tiles of the wave's columns from x0.
template <class T, int P>
__device__ __forceinline__ void add_to_r(f32x4 (&add)[P / 16], const Tile<T, P>& so, const Tile<T, P>& sq, const float* ut, int x0, int first, unsigned lane) {
    typedef BackChunk<T, P> C;
    const unsigned g = lane / 16, i16 = lane % 16;
#pragma unroll
    for (int et = 0; et < C::PT; et++) add[et] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int b = 0; b < C::LB; b++) {
        Frag<T> part[kParts<T>];
        scaled_parts(sq.down(b * 32, x0, lane), &ut[b * 32 + 8 * g], part);
#pragma unroll
        for (int et = 0; et < C::PT; et++) {
            const Frag<T> x = so.template down<true>(b * 32, acc_col(et), lane);
#pragma unroll
            for (int p = 0; p < kParts<T>; p++) mma(add[et], x, part[p]);
        }
    }
    float all = 0.f;
#pragma unroll
    for (int et = 0; et < C::PT; et++) watch(all, add[et]);
    if (!any_not_finite(all)) return;
#pragma unroll
    for (int et = 0; et < C::PT; et++) {
        add[et] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll 1
        for (int i = 0; i < first; i++)
#pragma unroll
            for (int r = 0; r < 4; r++)
                add[et][r] = fmaf(ut[i] * as_f32(*sq.at(i, x0 + i16)), as_f32(*so.at(i, acc_row(et, g, r))), add[et][r]);
    }
}

template <class T, int P>
__global__ void __launch_bounds__((BackChunk<T, P>::NT), 2) k_attend_back(MoAttend a, Cut cut) {
    typedef BackChunk<T, P> C;
    typedef HeadRows<T, C> Head;
    constexpr int L = C::L, K = C::K;
    extern __shared__ __align__(16) char lds[];
    BackLds<T, P>& s = *(BackLds<T, P>*)lds;
    const typename C::Rows sq{s.q}, sk{s.k}, sv{s.v}, so{s.o};
    const typename C::Scored sx(s.x);
    const int w = threadIdx.x / kWave;
    const int64_t nh = head_of_block(a.N * a.H), env = nh / a.H;
    if (nh >= a.N * a.H) return;
    const int h = (int)(nh % a.H), seg = blockIdx.y;
    const int64_t c0 = seg * cut.per_seg, c1 = min(c0 + cut.per_seg, cut.chunks);
    const int x0 = w * 16;     // the wave's rows of R and S, columns of dq and dk; of dv its columns
    const int64_t de = (int64_t)a.D * a.E;
    const Head q(a.q, env, h, a.D, a.D == P), k(a.k, env, h, a.D, a.D == P), v(a.v, env, h, a.E, a.E == P), o(a.dout, env, h, a.E, a.E == P);
    const Head dq(a.dq, env, h, a.D, on_pieces<T>(a.dq)), dk(a.dk, env, h, a.D, on_pieces<T>(a.dk)), dv(a.dv, env, h, a.E, on_pieces<T>(a.dv));
    const f32x4 zero = {0.f, 0.f, 0.f, 0.f};

    s.pw.fill(a.decay[h], a.scale);
    f32x4 R[C::PT];            // R^T: rows e, columns d
#pragma unroll
    for (int et = 0; et < C::PT; et++) R[et] = zero;
    const float* in = cut.segs > 1 ? cut.enter + ((int64_t)seg * a.N * a.H + nh) * de : a.dstate_out ? a.dstate_out + nh * de : nullptr;
    if (in) load_state<P, true>(a, in, x0, R);
    for (int64_t c = c1 - 1; c >= c0; c--) {
        const int64_t t0 = c * L;
        const int n = (int)min((int64_t)L, a.T - t0);
        __syncthreads();                                       // the last chunk's tiles are done with, its results in theirs
        q.bring(s.q, t0, n);
        k.bring(s.k, t0, n);
        v.bring(s.v, t0, n);
        o.bring(s.o, t0, n);
        if (c < c1 - 1) {
            const int n1 = (int)min((int64_t)L, a.T - t0 - L);
            dq.take(s.dq(), t0 + L, n1);
            dk.take(s.dk(), t0 + L, n1);
            dv.take(s.dv(), t0 + L, n1);
        }
        const unsigned lane = thread_here() % kWave, g = lane / 16, i16 = lane % 16;
        const uint64_t m = __ballot(start_of_lane(a, t0, n, env) != 0);
        const int last = seen_from(m, L - 1);
        if (threadIdx.x < L) {
            const int i = threadIdx.x;
            s.wt[i] = i < n && i >= last ? s.pw.pw[n - 1 - i] : 0.f;
            s.ut[i] = i < n && seen_from(m, i) < 0 ? a.scale * s.pw.pw[i + 1] : 0.f;
        }
        brought();

#pragma unroll
        for (int b = 0; b < C::PB; b++) {                      // R by rows d, for K R
            Frag<T> x[K];
            halves<T>(R[2 * b], R[2 * b + 1], x);
#pragma unroll
            for (int p = 0; p < K; p++)
#pragma unroll
                for (int j = 0; j < 8; j += C::Rows::EPV)
                    *(uint4*)typename C::Rows{s.r + p * P * P}.at(x0 + i16, b * 32 + 8 * g + j) = *(const uint4*)((const T*)&x[p] + j);
        }
        f32x4 bs[C::TPW];                                      // B, until A is done with
        const auto scores = [&](auto starts) {                 // A and B, a lane four neighbouring j of one i
#pragma unroll
            for (int z = 0; z < C::TPW; z++) {
                const int idx = w + z * C::WAVES;
                if (C::TILES % C::WAVES && idx >= C::TILES) break;
                int it, jt;
                C::score_tile(idx, it, jt);
                f32x4 x = zero, y = zero;
#pragma unroll
                for (int b = 0; b < C::PB; b++) {
                    mma(x, sk.along(jt * 16, b * 32, lane), sq.along(it * 16, b * 32, lane));
                    mma(y, sv.along(jt * 16, b * 32, lane), so.along(it * 16, b * 32, lane));
                }
                const int i = it * 16 + i16, j = jt * 16 + 4 * g, from = starts ? seen_from(m, i) : 0;
                const float* f = s.pw.sees(i, j);
#pragma unroll
                for (int r = 0; r < 4; r++) {
                    const bool sees = !starts || j + r >= from;
                    x[r] = sees ? x[r] * f[-r] : 0.f;
                    y[r] = sees ? y[r] * f[-r] : 0.f;
                }
                sx.put(i, j, x);
                bs[z] = y;
            }
        };
        if (m) scores(std::true_type{});
        else scores(std::false_type{});
        __syncthreads();

        // A result, transposed: a lane has four neighbouring columns of one step. own_of: the sum over the chunk's steps, the
        // scores times y's rows; far_of: what the entering state or its gradient adds, by a factor a step.
        const auto result = [&](auto put, const float* factor, auto far_of, auto own_of, bool down, const typename C::Rows& y) {
            const auto write = [&](int t, const f32x4& own, const f32x4& far) {
                const float f = factor[t * 16 + i16];
                f32x4 z;
#pragma unroll
                for (int r = 0; r < 4; r++) z[r] = fmaf(f, far[r], own[r]);
                if (m && f == 0.f) z = own;                    // (what is not seen may be anything)
                put(t, pack4(z, T{}));
            };
            float all = 0.f;
#pragma unroll
            for (int t = 0; t < C::LT; t++) {
                const f32x4 far = far_of(t), own = own_of(t);
                watch(all, own);
                write(t, own, far);
            }
            if (!any_not_finite(all)) return;
#pragma unroll 1
            for (int t = 0; t < C::LT; t++) {                  // over the steps j that step i sees (or that see it) of x_ij y_j
                const int i = t * 16 + i16, j0 = down ? i : max(seen_from(m, i), 0), j1 = down ? n - 1 : i;
                f32x4 own = zero;
#pragma unroll 1
                for (int j = j0; j <= j1 && (!down || seen_from(m, j) <= i); j++)
#pragma unroll
                    for (int r = 0; r < 4; r++) own[r] = fmaf(down ? sx.get(j, i) : sx.get(i, j), as_f32(*y.at(j, x0 + 4 * g + r)), own[r]);
                write(t, own, far_of(t));
            }
        };
        const auto to_tile = [&](T* tile) {
            return [=](int t, const Pack<T, 4>& z) { *(Pack<T, 4>*)typename C::Rows{tile}.at(t * 16 + i16, x0 + 4 * g) = z; };
        };
        const auto far_by = [&](const Frag<T> (&x)[C::PB][K], const typename C::Rows& rows) {
            return [&](int t) {
                f32x4 far = zero;
#pragma unroll
                for (int b = 0; b < C::PB; b++) {
                    const Frag<T> y = rows.along(t * 16, b * 32, lane);
#pragma unroll
                    for (int p = 0; p < K; p++) mma(far, x[b][p], y);
                }
                return far;
            };
        };
        const auto own_down = [&](const Frag<T> (&x)[C::LB]) { // over the steps from t's on
            return [&](int t) {
                f32x4 own = zero;
#pragma unroll
                for (int b = t / 2; b < C::LB; b++)
#pragma unroll
                    for (int p = 0; p < K; p++) mma(own, x[b], sx.part[p].down(b * 32, t * 16, lane));
                return own;
            };
        };

        // the state that enters the chunk: rows d of the wave, eight neighbouring columns e a lane (asked for here, used
        // after dV)
        f32x4 S[C::PB][2];
        {
            const int d = x0 + i16;
            if (c > 0) {
                const float* kept = (const float*)a.saved + (nh * (cut.chunks - 1) + c - 1) * (P * P) + d * P + 8 * g;
#pragma unroll
                for (int b = 0; b < C::PB; b++) {
                    S[b][0] = *(const f32x4*)(kept + b * 32);
                    S[b][1] = *(const f32x4*)(kept + b * 32 + 4);
                }
            } else {
#pragma unroll
                for (int b = 0; b < C::PB; b++)
#pragma unroll
                    for (int j = 0; j < 8; j++) {
                        const int e = b * 32 + 8 * g + j;
                        S[b][j / 4][j % 4] = a.state && d < a.D && e < a.E ? a.state[nh * de + d * a.E + e] : 0.f;
                    }
            }
        }

        Pack<T, 4> held[C::LT];                                // dV, until R's tiles are done with
        {
            Frag<T> of[C::LB], rf[C::PB][K];
#pragma unroll
            for (int b = 0; b < C::LB; b++) of[b] = so.down(b * 32, x0, lane);
#pragma unroll
            for (int b = 0; b < C::PB; b++)
#pragma unroll
                for (int p = 0; p < K; p++) rf[b][p] = typename C::Rows{s.r + p * P * P}.down(b * 32, x0, lane);
            result([&](int t, const Pack<T, 4>& z) {
#pragma unroll
                for (int u = 0; u < C::LT; u++)
                    if (u == t) held[u] = z;
            }, s.wt, far_by(rf, sk), own_down(of), true, so);
        }
        __syncthreads();                                       // A and R's tiles are done with
#pragma unroll
        for (int t = 0; t < C::LT; t++) to_tile(s.dv())(t, held[t]);
#pragma unroll
        for (int z = 0; z < C::TPW; z++) {
            const int idx = w + z * C::WAVES;
            if (C::TILES % C::WAVES && idx >= C::TILES) break;
            int it, jt;
            C::score_tile(idx, it, jt);
            sx.put(it * 16 + i16, jt * 16 + 4 * g, bs[z]);
        }
        __syncthreads();
        {
            Frag<T> kf[C::LB], sf[C::PB][K];
#pragma unroll
            for (int b = 0; b < C::LB; b++) kf[b] = sk.down(b * 32, x0, lane);
#pragma unroll
            for (int b = 0; b < C::PB; b++) halves<T>(S[b][0], S[b][1], sf[b]);
            result(to_tile(s.dq()), s.ut, far_by(sf, so), [&](int t) {
                f32x4 own = zero;
#pragma unroll
                for (int b = 0; b <= t / 2; b++)
#pragma unroll
                    for (int p = 0; p < K; p++) mma(own, kf[b], sx.part[p].along(t * 16, b * 32, lane));
                return own;
            }, false, sk);
        }
        {
            Frag<T> qf[C::LB], rf[C::PB][K];
#pragma unroll
            for (int b = 0; b < C::LB; b++) qf[b] = sq.down(b * 32, x0, lane);
#pragma unroll
            for (int b = 0; b < C::PB; b++) halves<T>(R[2 * b], R[2 * b + 1], rf[b]);
            result(to_tile(s.dk()), s.wt, far_by(rf, sv), own_down(qf), true, sq);
        }

        f32x4 add[C::PT];                                      // R'
        add_to_r<T, P>(add, so, sq, s.ut, x0, m ? (int)__ffsll((long long)m) - 1 : n, lane);
        const float f = s.pw.pw[n];
#pragma unroll
        for (int et = 0; et < C::PT; et++)
#pragma unroll
            for (int r = 0; r < 4; r++) R[et][r] = m ? add[et][r] : fmaf(f, R[et][r], add[et][r]);
    }
    if (c0 < c1) {
        __syncthreads();
        const int n = (int)min((int64_t)L, a.T - c0 * L);
        dq.take(s.dq(), c0 * L, n);
        dk.take(s.dk(), c0 * L, n);
        dv.take(s.dv(), c0 * L, n);
    }
    if (a.dstate && cut.segs == 1) store_state<P, true>(a, a.dstate + nh * de, x0, R);
}

// A segment's own sum of R' (see R' above) and what it leaves of a gradient that comes from behind it.
template <class T, int P>
__global__ void __launch_bounds__((BackChunk<T, P>::NT)) k_attend_back_sums(MoAttend a, Cut cut) {
    typedef BackChunk<T, P> C;
    typedef HeadRows<T, C> Head;
    constexpr int L = C::L;
    __shared__ __align__(16) T lq[L * P], lo[L * P];
    __shared__ Powers<L> pw;
    __shared__ __align__(16) float ut[L];
    const typename C::Rows sq{lq}, so{lo};
    const int64_t nh = head_of_block(a.N * a.H), env = nh / a.H;
    if (nh >= a.N * a.H) return;
    const int h = (int)(nh % a.H), seg = blockIdx.y;
    const int64_t c0 = seg * cut.per_seg, c1 = min(c0 + cut.per_seg, cut.chunks);
    const int x0 = threadIdx.x / kWave * 16;
    const Head q(a.q, env, h, a.D, a.D == P), o(a.dout, env, h, a.E, a.E == P);
    pw.fill(a.decay[h], a.scale);
    f32x4 R[C::PT];
#pragma unroll
    for (int et = 0; et < C::PT; et++) R[et] = f32x4{0.f, 0.f, 0.f, 0.f};
    bool any_start = false;
    for (int64_t c = c1 - 1; c >= c0; c--) {
        const int64_t t0 = c * L;
        const int n = (int)min((int64_t)L, a.T - t0);
        __syncthreads();
        q.bring(lq, t0, n);
        o.bring(lo, t0, n);
        const uint64_t m = __ballot(start_of_lane(a, t0, n, env) != 0);
        any_start |= m != 0;
        if (threadIdx.x < L) ut[threadIdx.x] = (int)threadIdx.x < n && seen_from(m, threadIdx.x) < 0 ? a.scale * pw.pw[threadIdx.x + 1] : 0.f;
        brought();
        f32x4 add[C::PT];
        add_to_r<T, P>(add, so, sq, ut, x0, m ? (int)__ffsll((long long)m) - 1 : n, thread_here() % kWave);
        const float f = pw.pw[n];
#pragma unroll
        for (int et = 0; et < C::PT; et++)
#pragma unroll
            for (int r = 0; r < 4; r++) R[et][r] = m ? add[et][r] : fmaf(f, R[et][r], add[et][r]);
    }
    float* to = cut.enter + ((int64_t)seg * a.N * a.H + nh) * a.D * a.E;
    store_state<P, true>(a, to, x0, R);
    if (threadIdx.x == 0) {
        const int64_t n = min(c1 * L, a.T) - c0 * L;
        cut.keep[(int64_t)seg * a.N * a.H + nh] = any_start ? -1.f : power(a.decay[h], n);
    }
}

template <class T, int P> int attend_back_chunks(const MoAttend& a, hipStream_t s) {
    Cut c = attend_cut(a);
    cut_place(a, c);
    static_assert(sizeof(BackLds<T, P>) <= (160 << 10), "");
    const dim3 grid = grid_of(a.N * a.H, c.segs), block(BackChunk<T, P>::NT);
    if (c.segs > 1) {
        hipLaunchKernelGGL((k_attend_back_sums<T, P>), grid, block, 0, s, a, c);
        if (launched("k_attend_back_sums") || enter_states(a, c, a.dstate_out, a.dstate, true, s)) return -1;
    }
    hipLaunchKernelGGL((k_attend_back<T, P>), grid, block, sizeof(BackLds<T, P>), s, a, c);
    return launched("k_attend_back");
}

}  // namespace mo
