// The gradient of the selective state space scan.
#pragma once
#include "scan.hpp"

namespace mo {

// Back through the chunks from the states kept before each: a chunk's states are made again and stay in registers, then the steps go
// backwards with Q, the gradient of the state after a step from all later ones:
//   R = C dy + Q,  dC = sum_c h dy,  dB = sum_c R u,  du = sum_s R B,  q = R a h_{t-1},  dA += q d,  dd = du x + sum_s q A,  Q = R a
// (u = d x, a = exp(d A), 0 where the episode starts). The sums over channels are joined in the wave (wave_sums) and leave as one row a wave.
// SUMS: only what a segment adds to the Q that comes out of it, and the sum of its step sizes.
template <class T, int SP, bool SPLIT, bool SUMS>
__global__ void __launch_bounds__(SCAN_WAVES* kWave) k_scan_back(Scan k) {
    const MoScan& a = k.a;
    __shared__ float part[SPLIT ? SCAN_WAVES : 1][SPLIT ? SCAN_STEPS : 1][3][kWave];
    __shared__ float ends[SPLIT ? SCAN_WAVES : 1][2][kWave];
    const int w = wave_here(), slice = SPLIT ? w : 0;
    const int64_t wave = SPLIT ? block_here() : block_here() * SCAN_WAVES + w;
    const int64_t items = k.segments * a.N, cbs = a.G * k.per, at_once = SUMS ? items : k.rows;
    if (wave >= at_once * cbs) return;
    float A[SP], dA[SP], dD = 0.f, dbias = 0.f;
    {
        const ScanPlace me(k, wave, slice, SP);
        load_decays<SP>(a, me.c, me.s0, A);
    }
#pragma unroll
    for (int s = 0; s < SP; s++) dA[s] = 0.f;
    for (int64_t item = wave / cbs; item < items; item += at_once) {
        const ScanPlace me(k, item * cbs + wave % cbs, slice, SP);
        const int64_t n = me.n, first = me.segment * k.each, last = min(k.chunks, first + k.each);
        const int c = me.c;
        const float bias = a.dt_bias ? a.dt_bias[c] : 0.f, D = a.D ? a.D[c] : 0.f;
        const int64_t seg0 = ((me.segment * a.N + n) * k.SB + me.s0) * a.C + c;
        float Q[SP], total = 0.f;
#pragma unroll
        for (int s = 0; s < SP; s++) {
            if (SUMS) Q[s] = 0.f;
            else if (k.segments > 1) Q[s] = k.seg_h[seg0 + (int64_t)s * a.C];
            else Q[s] = a.dstate_out && me.s0 + s < a.S ? a.dstate_out[(n * a.C + c) * a.S + me.s0 + s] : 0.f;
        }
        // a step's inputs that are not the states'
        struct In { float x, d, slope, z, sig, dout, dy; };
        const auto inputs = [&](int64_t t) {
            In v;
            const Size p = softplus(at_row<T>(a.dt, t, n, c) + bias);
            v.x = SUMS ? 0.f : at_row<T>(a.x, t, n, c);
            v.d = p.d;
            v.slope = p.slope;
            v.dout = me.live ? at_row<T>(a.dout, t, n, c) : 0.f;    // (an idle lane adds nothing to dB and dC)
            v.z = v.sig = v.dy = 0.f;
            if (a.z.p) {
                v.z = at_row<T>(a.z, t, n, c);
                v.sig = sigmoid(v.z);
                v.dy = v.dout * (v.z * v.sig);
            } else {
                v.dy = v.dout;
            }
            return v;
        };
        const auto finish = [&](int64_t t, const In& v, float y, float du, float dd) {
            const float ddt = fmaf(du, v.x, dd * LN2) * v.slope;
            dD = fmaf(v.dy, v.x, dD);
            dbias += ddt;
            if (!me.live) return;
            to_row<T>(a.dx, t, n, c, fmaf(du, v.d, D * v.dy));
            to_row<T>(a.ddt, t, n, c, ddt);
            if (a.z.p) to_row<T>(a.dz, t, n, c, v.dout * fmaf(D, v.x, y) * (v.sig * fmaf(v.z, 1.f - v.sig, 1.f)));
        };
        for (int64_t chunk = last - 1; chunk >= first; chunk--) {
            const int64_t t0 = chunk * SCAN_STEPS;
            const int steps = (int)min((int64_t)SCAN_STEPS, a.T - t0);
            const unsigned cuts = starts_from(a, t0, steps, n, me.lane);
            const auto row_of = [&](int64_t t) { return (t * a.N + n) * a.G + me.g; };
            float h[SUMS ? 1 : SCAN_STEPS + 1][SP];
            if (!SUMS) {
                const float* from = k.kept + ((chunk * a.N + n) * k.SB + me.s0) * a.C + c;
#pragma unroll
                for (int s = 0; s < SP; s++) h[0][s] = from[(int64_t)s * a.C];
#pragma unroll
                for (int i = 0; i < SCAN_STEPS; i++) {
                    if (i >= steps) break;
                    const int64_t t = t0 + i;
                    const float d = softplus(at_row<T>(a.dt, t, n, c) + bias).d, u = d * at_row<T>(a.x, t, n, c);
                    const Uniform B = uniform(k.bc + row_of(t) * 2 * k.SB + me.s0);
                    const bool cut = cuts >> i & 1;
#pragma unroll
                    for (int s = 0; s < SP; s++) {
                        const float add = u * B[s];
                        h[SUMS ? 0 : i + 1][s] = cut ? add : fmaf(exp2_raw(d * A[s]), h[SUMS ? 0 : i][s], add);
                    }
                }
            }
#pragma unroll
            for (int i = SCAN_STEPS - 1; i >= 0; i--) {
                if (i >= steps) continue;
                const int64_t t = t0 + i;
                const In v = inputs(t);
                const Uniform B = uniform(k.bc + row_of(t) * 2 * k.SB + me.s0), C = B + k.SB;
                const bool cut = cuts >> i & 1;
                if constexpr (SUMS) {
#pragma unroll
                    for (int s = 0; s < SP; s++) Q[s] = fmaf(C[s], v.dy, Q[s]) * exp2_raw(v.d * A[s]);
                    if (cut) {
#pragma unroll
                        for (int s = 0; s < SP; s++) Q[s] = 0.f;
                        total = -1.f;
                    }
                    if (total >= 0.f) total += v.d;
                } else {
                    const float u = v.d * v.x;
                    float y = 0.f, du = 0.f, dd = 0.f, sums[2 * SP];
#pragma unroll
                    for (int s = 0; s < SP; s++) {
                        const float R = fmaf(C[s], v.dy, Q[s]);
                        y = fmaf(C[s], h[i + 1][s], y);
                        sums[s] = me.live ? R * u : 0.f;
                        sums[SP + s] = me.live ? h[i + 1][s] * v.dy : 0.f;
                        du = fmaf(R, B[s], du);
                        Q[s] = R * exp2_raw(v.d * A[s]);
                    }
                    if (cut) {
#pragma unroll
                        for (int s = 0; s < SP; s++) Q[s] = 0.f;
                    } else {
#pragma unroll
                        for (int s = 0; s < SP; s++) {
                            const float q = Q[s] * h[i][s];
                            dd = fmaf(q, A[s], dd);
                            dA[s] = fmaf(q, v.d, dA[s]);
                        }
                    }
                    const float sum = wave_sums<2 * SP>(sums);
                    const int slot = sum_slot(me.lane, 2 * SP);
                    if (slot < 2 * SP) {
                        const int64_t cb = wave % cbs % k.per;
                        k.part_bc[(cb * a.T * a.N * a.G + row_of(t)) * 2 * k.SB + (slot < SP ? 0 : k.SB - SP) + me.s0 + slot] = sum;
                    }
                    if (SPLIT) {
                        part[slice][i][0][me.lane] = y;
                        part[slice][i][1][me.lane] = du;
                        part[slice][i][2][me.lane] = dd;
                    } else {
                        finish(t, v, y, du, dd);
                    }
                }
            }
            if (SPLIT && !SUMS) {
                __syncthreads();
                for (int i = slice; i < steps; i += k.slices) {
                    float j[3] = {0.f, 0.f, 0.f};
                    for (int s = 0; s < k.slices; s++)
                        for (int m = 0; m < 3; m++) j[m] += part[s][i][m][me.lane];
                    finish(t0 + i, inputs(t0 + i), j[0], j[1], j[2]);
                }
                __syncthreads();
            }
        }
        if (!me.live) continue;
        if (SUMS) {
#pragma unroll
            for (int s = 0; s < SP; s++) k.seg_h[seg0 + (int64_t)s * a.C] = Q[s];
            if (slice == 0) k.seg_d[(me.segment * a.N + n) * a.C + c] = total;
        } else if (first == 0 && a.dstate) {
#pragma unroll
            for (int s = 0; s < SP; s++)
                if (me.s0 + s < a.S) a.dstate[(n * a.C + c) * a.S + me.s0 + s] = Q[s];
        }
    }
    if (SUMS) return;
    if (SPLIT) {
        ends[slice][0][threadIdx.x % kWave] = dD;
        ends[slice][1][threadIdx.x % kWave] = dbias;
        __syncthreads();
        dD = dbias = 0.f;
        for (int s = 0; s < k.slices; s++) {
            dD += ends[s][0][threadIdx.x % kWave];
            dbias += ends[s][1][threadIdx.x % kWave];
        }
    }
    const ScanPlace me(k, wave, slice, SP);
    if (!me.live) return;
    float* to = k.part + wave / cbs * (k.SB + 2) * a.C + me.c;
#pragma unroll
    for (int s = 0; s < SP; s++) to[(int64_t)(me.s0 + s) * a.C] = dA[s];
    if (slice == 0) {
        to[(int64_t)k.SB * a.C] = dD;
        to[(int64_t)(k.SB + 1) * a.C] = dbias;
    }
}

// dB and dC from the rows that the waves of a group's channels left.
template <class T> __global__ void __launch_bounds__(256) k_scan_join(Scan k) {
    const MoScan& a = k.a;
    const int64_t rows = a.T * a.N * a.G, id = block_here() * 256 + threadIdx.x, row = id / (2 * k.SB);
    if (row >= rows) return;
    const int i = (int)(id % (2 * k.SB)), s = i % k.SB, g = (int)(row % a.G);
    if (s >= a.S) return;
    float x = 0.f;
    for (int p = 0; p < k.per; p++) x += k.part_bc[p * rows * 2 * k.SB + id];
    const int64_t n = row / a.G % a.N, t = row / a.G / a.N;
    const MoRows& r = i < k.SB ? a.dB : a.dC;
    ((T*)r.p)[t * r.st + n * r.sn + g * r.sh + s] = as<T>(x);
}

template <class T> int scan_backward(const MoScan& a, hipStream_t s) {
    Scan k = scan_cut(a, true);
    k.bc = (const float*)a.saved;
    k.kept = (float*)a.saved + scan_bc(k);
    k.seg_h = (float*)a.work;
    k.seg_d = k.seg_h + k.segments * a.N * k.SB * a.C;
    k.part_bc = (float*)a.work + scan_segs(k);
    k.part = k.part_bc + scan_parts_bc(k);
    float* more = k.part + scan_parts(k);
    return by_states(k, [&](auto sp, auto split) {
        constexpr int SP = decltype(sp)::value;
        constexpr bool SPLIT = decltype(split)::value;
        dim3 grid, block;
        if (k.segments > 1) {
            scan_launch_shape(k, k.segments * a.N * a.G * k.per, grid, block);
            hipLaunchKernelGGL((k_scan_back<T, SP, SPLIT, true>), grid, block, 0, s, k);
            hipLaunchKernelGGL((k_scan_enter<true>), grid_of((a.N * k.SB * a.C + 255) / 256), dim3(256), 0, s, k);
        }
        scan_launch_shape(k, k.rows * a.G * k.per, grid, block);
        hipLaunchKernelGGL((k_scan_back<T, SP, SPLIT, false>), grid, block, 0, s, k);
        if (launched("k_scan_back")) return -1;
        const int64_t n = a.T * a.N * a.G * 2 * k.SB;
        if (n) hipLaunchKernelGGL((k_scan_join<T>), grid_of((n + 255) / 256), dim3(256), 0, s, k);
        if (launched("k_scan_join")) return -1;
        if (!a.dA && !a.dD && !a.ddt_bias) return 0;
        return column_sums(ColumnSums{k.part, more, k.rows, k.SB + 2, a.C, a.S, k.SB, a.dA, a.dD, a.ddt_bias}, s);
    });
}

}  // namespace mo
