// The gradient of the selective state space scan.
#pragma once
#include "scan.hpp"

namespace mo {

// Back through the chunks from the states kept before each: a chunk's states are made again and stay in registers, then the steps go
// backwards with Q, the gradient of the state after a step from all later ones:
//   R = C dy + Q,  dC = sum_c h dy,  dB = sum_c R u,  du = sum_s R B,  Q = R a,  q = Q h_{t-1},  dA += q d,  dd = du x + sum_s q A
// (u = d x, a = exp(d A); Q and q are 0 where the episode starts). The sums over channels are joined in the wave (wave_sums), then in LDS over the
// workgroup's waves, which have neighbouring channels of one env and segment.
constexpr int BACK_WAVES = SCAN_BACK_WAVES;

// Where bit I of cuts is set: x = y = 0, for all states.
template <int I, int SP> __device__ __forceinline__ void if_start_clear(unsigned cuts, float (&x)[SP], float (&y)[SP]) {
#pragma unroll
    for (int s = 0; s < SP; s += 4)
        asm volatile(
            "s_bitcmp1_b32 %[m], %[i]\n\ts_cbranch_scc0 .Lstart%=\n\tv_mov_b32 %0, 0\n\tv_mov_b32 %1, 0\n\tv_mov_b32 %2, 0\n\tv_mov_b32 %3, 0\n\t"
            "v_mov_b32 %4, 0\n\tv_mov_b32 %5, 0\n\tv_mov_b32 %6, 0\n\tv_mov_b32 %7, 0\n.Lstart%=:"
            : "+v"(x[s]), "+v"(x[s + 1]), "+v"(x[s + 2]), "+v"(x[s + 3]), "+v"(y[s]), "+v"(y[s + 1]), "+v"(y[s + 2]), "+v"(y[s + 3])
            : [m] "s"(cuts), [i] "n"(I)
            : "scc");
}

// What a segment adds to the Q that comes out of it, and the sum of its step sizes (-1 where an episode starts in it).
template <class T, int SP, bool SPLIT>
__global__ void __launch_bounds__(SCAN_WAVES* kWave) k_scan_back_sums(Scan k) {
    const MoScan& a = k.a;
    constexpr int TILE = SCAN_STEPS * kWave;
    __shared__ __attribute__((aligned(16))) T tiles[SCAN_WAVES][3][TILE];
    const int w = wave_here(), slice = SPLIT ? w : 0, cbs = a.G * k.per;
    const int64_t wave = SPLIT ? block_here() : block_here() * SCAN_WAVES + w;
    if (wave >= k.segments * a.N * cbs) return;
    const ScanPlace me(k, wave / cbs, (int)(wave % cbs), slice, SP);
    const int64_t n = me.n, first = me.segment * k.each, last = min(k.chunks, first + k.each);
    const int lane = me.lane;
    T *ldo = tiles[w][0], *ldt = tiles[w][1], *lz = tiles[w][2];
    const bool gate = a.z.p;
    float A[SP], Q[SP], total = 0.f;
    load_decays<SP>(a, me, A);
#pragma unroll
    for (int s = 0; s < SP; s++) Q[s] = 0.f;
    const float bias = a.dt_bias ? a.dt_bias[me.c] : 0.f;
    ChunkIn<T> ido, idt, iz;
    uint8_t flag = 0;
    const auto steps_of = [&](int64_t chunk) { return (int)min((int64_t)SCAN_STEPS, a.T - chunk * SCAN_STEPS); };
    const auto ahead = [&](int64_t chunk) {
        const int64_t t0 = chunk * SCAN_STEPS;
        const int steps = steps_of(chunk);
        flag = start_of_lane(a, t0, steps, me);
        if (!k.wide) return;
        ido.ahead(a.dout, t0, steps, me);
        idt.ahead(a.dt, t0, steps, me);
        if (gate) iz.ahead(a.z, t0, steps, me);
    };
    ahead(last - 1);
    const int64_t bc_step = a.N * a.G * 2 * k.SB;
    Uniform bc = uniform(k.bc + ((last * SCAN_STEPS * a.N + n) * a.G + me.g) * 2 * k.SB + k.SB + me.s0) - bc_step;
    float now[SP];
#pragma unroll
    for (int s = 0; s < SP; s++) now[s] = bc[s];
    for (int64_t chunk = last - 1; chunk >= first; chunk--) {
        const int64_t t0 = chunk * SCAN_STEPS;
        const int steps = steps_of(chunk);
        const unsigned cuts = (unsigned)__ballot(flag != 0);
        wave_wrote();
        if (k.wide) {
            ido.arrive(ldo, steps, me);
            idt.arrive(ldt, steps, me, NO_SIZE<T>);
            if (gate) iz.arrive(lz, steps, me);
        } else {
            ChunkIn<T>::narrow(ldo, a.dout, t0, steps, me);
            ChunkIn<T>::narrow(ldt, a.dt, t0, steps, me, -INFINITY);
            if (gate) ChunkIn<T>::narrow(lz, a.z, t0, steps, me);
        }
        wave_wrote();
        if (chunk > first) ahead(chunk - 1);
        float d[SCAN_STEPS], dy[SCAN_STEPS];
#pragma unroll
        for (int i = 0; i < SCAN_STEPS; i++) {
            d[i] = softplus(as_f32(ldt[i * kWave + lane]) + bias).d;
            dy[i] = as_f32(ldo[i * kWave + lane]);
            if (gate) {
                const float z = as_f32(lz[i * kWave + lane]);
                dy[i] *= z * sigmoid(z);
            }
            total = cuts >> i & 1 || total < 0.f ? -1.f : total + d[i];
        }
        end_of_step();
        each_step([&](auto step) {
            constexpr int i = SCAN_STEPS - 1 - decltype(step)::value;
            float next[SP], zero[SP];
            bc = move_on(bc, i || chunk ? -bc_step : 0);      // (there is no step before the first)
#pragma unroll
            for (int s = 0; s < SP; s++) next[s] = bc[s];
#pragma unroll
            for (int s = 0; s < SP; s++) {
                Q[s] = fmaf(now[s], dy[i], Q[s]) * exp2_raw(d[i] * A[s]);
                zero[s] = 0.f;
            }
            if_start_set<i, SP>(cuts, Q, 0.f, zero);
#pragma unroll
            for (int s = 0; s < SP; s++) now[s] = next[s];
            end_of_step();
        });
    }
    if (!me.live) return;
#pragma unroll
    for (int s = 0; s < SP; s++) k.seg_h[((me.segment * a.N + n) * k.SB + me.s0 + s) * a.C + me.c] = Q[s];
    if (slice == 0) k.seg_d[(me.segment * a.N + n) * a.C + me.c] = total;
}

// Workgroups of `wide` waves of channels by `slices`; LDS is a wave's own tiles of x, dt, z and dout (whose places dx, ddt and dz take), its
// step sizes, and the sums for its workgroup's dB and dC, of two chunks in turn.
template <class T> constexpr int back_wave_lds() { return 4 * SCAN_STEPS * kWave * (int)sizeof(T) + SCAN_STEPS * kWave * 4 + 2 * SCAN_STEPS * 32 * 4; }

template <class T, int SP, bool SPLIT>
__global__ void __launch_bounds__(BACK_WAVES* kWave, 2) k_scan_back(Scan k) {
    const MoScan& a = k.a;
    constexpr int TILE = SCAN_STEPS * kWave;
    extern __shared__ __attribute__((aligned(16))) char lds[];
    __shared__ float part[SPLIT ? BACK_WAVES : 1][SPLIT ? SCAN_STEPS : 1][SPLIT ? 3 : 1][kWave];
    const int w = wave_here(), slices = SPLIT ? k.slices : 1, slice = SPLIT ? w % slices : 0, across = w / slices;
    const int64_t items = k.segments * a.N, row = block_here() / (a.G * k.cuts), bg = block_here() % (a.G * k.cuts);
    if (row >= k.rows) return;
    const int g0 = (int)(bg / k.cuts), cut = (int)(bg % k.cuts), in_group = cut * k.across + across;   // (waves past the group's channels join the barriers only)
    const int cb = g0 * k.per + min(in_group, k.per - 1);
    const bool idle = in_group >= k.per;
    T* lx = (T*)(lds + w * back_wave_lds<T>());
    T *ldt = lx + TILE, *lz = lx + 2 * TILE, *ldo = lx + 3 * TILE;
    float *ld = (float*)(lx + 4 * TILE), *sums = ld + TILE;                // (2, SCAN_STEPS, 32)
    const bool gate = a.z.p;
    ScanPlace me(k, row, cb, slice, SP);
    if (idle) { me.live = false; me.there = 0; }
    const int lane = me.lane, c = me.c;
    float A[SP], dA[SP], dD = 0.f, dbias = 0.f;
    load_decays<SP>(a, me, A);
    const float bias = a.dt_bias ? a.dt_bias[c] : 0.f, D = a.D ? a.D[c] : 0.f;
#pragma unroll
    for (int s = 0; s < SP; s++) dA[s] = 0.f;
    const auto steps_of = [&](int64_t chunk) { return (int)min((int64_t)SCAN_STEPS, a.T - chunk * SCAN_STEPS); };
    const int64_t bc_step = a.N * a.G * 2 * k.SB;
    for (int64_t item = row; item < items; item += k.rows) {
        const int64_t n = me.n = item % a.N;
        me.segment = item / a.N;
        const int64_t first = me.segment * k.each, last = min(k.chunks, first + k.each);
        float Q[SP], before[SP];
        ChunkIn<T> ix, idt, iz, ido;
        uint8_t flag = 0;
        const auto ahead = [&](int64_t chunk) {
            const int64_t t0 = chunk * SCAN_STEPS;
            const int steps = steps_of(chunk);
            flag = start_of_lane(a, t0, steps, me);
            const float* from = k.kept + ((chunk * a.N + n) * k.SB + me.s0) * a.C + c;
#pragma unroll
            for (int s = 0; s < SP; s++) before[s] = __builtin_nontemporal_load(from + (int64_t)s * a.C);
            if (!k.wide) return;
            ix.ahead(a.x, t0, steps, me);
            idt.ahead(a.dt, t0, steps, me);
            if (gate) iz.ahead(a.z, t0, steps, me);
            ido.ahead(a.dout, t0, steps, me);
        };
        if (first < last) ahead(last - 1);
#pragma unroll
        for (int s = 0; s < SP; s++) {
            if (!me.live) Q[s] = 0.f;
            else if (k.segments > 1) Q[s] = k.seg_h[((me.segment * a.N + n) * k.SB + me.s0 + s) * a.C + c];
            else Q[s] = a.dstate_out && me.s0 + s < a.S ? a.dstate_out[(n * a.C + c) * a.S + me.s0 + s] : 0.f;
        }
        for (int64_t chunk = last - 1; chunk >= first; chunk--) {
            const int64_t t0 = chunk * SCAN_STEPS;
            const int steps = steps_of(chunk);
            const unsigned cuts = (unsigned)__ballot(flag != 0);
            float h[SCAN_STEPS + 1][SP];
#pragma unroll
            for (int s = 0; s < SP; s++) h[0][s] = me.live ? before[s] : 0.f;
            wave_wrote();
            if (k.wide) {
                ix.arrive(lx, steps, me);
                idt.arrive(ldt, steps, me, NO_SIZE<T>);
                if (gate) iz.arrive(lz, steps, me);
                ido.arrive(ldo, steps, me);
            } else {
                ChunkIn<T>::narrow(lx, a.x, t0, steps, me);
                ChunkIn<T>::narrow(ldt, a.dt, t0, steps, me, -INFINITY);
                if (gate) ChunkIn<T>::narrow(lz, a.z, t0, steps, me);
                ChunkIn<T>::narrow(ldo, a.dout, t0, steps, me);
            }
            wave_wrote();
            Uniform bc = uniform(k.bc + ((t0 * a.N + n) * a.G + g0) * 2 * k.SB + me.s0);
            {   // the states again
                float d[SCAN_STEPS], u[SCAN_STEPS];
#pragma unroll
                for (int i = 0; i < SCAN_STEPS; i++) {
                    d[i] = softplus(as_f32(ldt[i * kWave + lane]) + bias).d;
                    u[i] = d[i] * as_f32(lx[i * kWave + lane]);
                    ld[i * kWave + lane] = d[i];
                }
                StepBC<SP> now;
                load_bc<SP, false>(now, bc, k.SB);
                end_of_step();
                each_step([&](auto step) {
                    constexpr int i = decltype(step)::value;
                    StepBC<SP> next;
                    if constexpr (i + 1 < SCAN_STEPS) {
                        bc = move_on(bc, bc_step);
                        load_bc<SP, false>(next, bc, k.SB);
                    }
#pragma unroll
                    for (int s = 0; s < SP; s++) h[i + 1][s] = fmaf(exp2_raw(d[i] * A[s]), h[i][s], u[i] * now.b[s]);
                    if_start_set<i, SP>(cuts, h[i + 1], u[i], now.b);
                    if constexpr (i + 1 < SCAN_STEPS) now = next;
                    end_of_step();
                });
            }
            float* const to_join = sums + (chunk & 1) * SCAN_STEPS * 32;
            const int slot = sum_slot(lane, 2 * SP);
            StepBC<SP> now;
            load_bc<SP>(now, bc, k.SB);
            each_step([&](auto step) {
                constexpr int i = SCAN_STEPS - 1 - decltype(step)::value;
                const int at = i * kWave + lane;
                const float x = as_f32(lx[at]), dout = as_f32(ldo[at]), d = ld[at], z = gate ? as_f32(lz[at]) : 0.f, raw = as_f32(ldt[at]) + bias;
                const float sig = sigmoid(z), dy = gate ? dout * (z * sig) : dout, u = d * x;
                StepBC<SP> next;
                float y = 0.f, du = 0.f, dd = 0.f, q[SP], v[SP];
#pragma unroll
                for (int s = 0; s < SP; s++) {
                    y = fmaf(now.c[s], h[i + 1][s], y);
                    v[s] = h[i + 1][s] * dy;
                }
                float sum_c = wave_sums<SP>(v);
                made(y);
                made(sum_c);
                end_of_step();
#pragma unroll
                for (int s = 0; s < SP; s++) {
                    Q[s] = fmaf(now.c[s], dy, Q[s]);
                    du = fmaf(Q[s], now.b[s], du);
                    v[s] = Q[s] * u;
                }
                made(du);
                if constexpr (i > 0) {
                    bc = move_on(bc, -bc_step);
                    load_bc<SP>(next, bc, k.SB);
                }
                float sum_b = wave_sums<SP>(v);
                made(sum_b);
                end_of_step();
#pragma unroll
                for (int s = 0; s < SP; s++) {
                    Q[s] *= exp2_raw(d * A[s]);
                    q[s] = Q[s] * h[i][s];
                }
                if_start_clear<i, SP>(cuts, Q, q);
#pragma unroll
                for (int s = 0; s < SP; s++) {
                    dd = fmaf(q[s], A[s], dd);
                    dA[s] = fmaf(q[s], d, dA[s]);
                }
                if (slot < SP) to_join[i * 32 + slot + (lane & 1 ? SP : 0)] = lane & 1 ? sum_c : sum_b;
                if constexpr (SPLIT) {
                    part[w][i][0][lane] = y;
                    part[w][i][1][lane] = du;
                    part[w][i][2][lane] = dd;
                } else {
                    const float slope = softplus(raw).slope, ddt = fmaf(du, x, dd * LN2) * slope;
                    dD = fmaf(dy, x, dD);
                    dbias += ddt;
                    lx[at] = as<T>(fmaf(du, d, D * dy));
                    ldt[at] = as<T>(ddt);
                    if (gate) lz[at] = as<T>(dout * fmaf(D, x, y) * (sig * fmaf(z, 1.f - sig, 1.f)));
                }
                if constexpr (i > 0) now = next;
                if constexpr (i == SCAN_STEPS / 2) {
                    if (chunk > first) ahead(chunk - 1);      // (the states that are done with have left their registers)
                }
                end_of_step();
            });
            __syncthreads();
            if constexpr (SPLIT) {
                for (int i = slice; i < steps; i += slices) {
                    const int at = i * kWave + lane;
                    const float x = as_f32(lx[at]), dout = as_f32(ldo[at]), d = ld[at], z = gate ? as_f32(lz[at]) : 0.f;
                    const float sig = sigmoid(z), dy = gate ? dout * (z * sig) : dout, slope = softplus(as_f32(ldt[at]) + bias).slope;
                    float j[3] = {0.f, 0.f, 0.f};
                    for (int s = 0; s < slices; s++)
#pragma unroll
                        for (int m = 0; m < 3; m++) j[m] += part[w - slice + s][i][m][lane];
                    const float ddt = fmaf(j[1], x, j[2] * LN2) * slope;
                    dD = fmaf(dy, x, dD);
                    dbias += ddt;
                    if (!me.live) continue;
                    const auto row_of = [&](const MoRows& r) { return (T*)r.p + (t0 + i) * r.st + n * r.sn + c; };
                    *row_of(a.dx) = as<T>(fmaf(j[1], d, D * dy));
                    *row_of(a.ddt) = as<T>(ddt);
                    if (gate) *row_of(a.dz) = as<T>(dout * fmaf(D, x, j[0]) * (sig * fmaf(z, 1.f - sig, 1.f)));
                }
            } else {
                ChunkIn<T>::leave(lx, a.dx, t0, steps, me, k.wide);
                ChunkIn<T>::leave(ldt, a.ddt, t0, steps, me, k.wide);
                if (gate) ChunkIn<T>::leave(lz, a.dz, t0, steps, me, k.wide);
            }
            // dB and dC of the chunk: the workgroup's waves joined (the next chunk's sums go to the other place)
            for (int i = threadIdx.x; i < steps * 2 * k.SB; i += blockDim.x) {
                const int j = i / (2 * k.SB), m = i % (2 * k.SB), which = m / k.SB, s = m % k.SB, of = s / SP;
                float x = 0.f;
                for (int v = of; v < k.across * slices; v += slices)
                    x += ((float*)(lds + v * back_wave_lds<T>() + 4 * TILE * sizeof(T)) + TILE)[(chunk & 1) * SCAN_STEPS * 32 + j * 32 + which * SP + s % SP];
                if (k.cuts > 1) {
                    k.part_bc[((((int64_t)cut * a.T + t0 + j) * a.N + n) * a.G + g0) * 2 * k.SB + m] = x;
                } else if (s < a.S) {
                    const MoRows& r = which ? a.dC : a.dB;
                    ((T*)r.p)[(t0 + j) * r.st + n * r.sn + g0 * r.sh + s] = as<T>(x);
                }
            }
            if constexpr (SPLIT) __syncthreads();             // (their partial sums have been read)
        }
        if (first == 0 && a.dstate && me.live)
#pragma unroll
            for (int s = 0; s < SP; s++)
                if (me.s0 + s < a.S) a.dstate[(n * a.C + c) * a.S + me.s0 + s] = Q[s];
        __syncthreads();                                      // (one env's last sums are read before the next one's first)
    }
    if constexpr (SPLIT) {
        part[w][0][0][lane] = dD;
        part[w][0][1][lane] = dbias;
        __syncthreads();
        dD = dbias = 0.f;
        for (int s = 0; s < slices; s++) {
            dD += part[w - slice + s][0][0][lane];
            dbias += part[w - slice + s][0][1][lane];
        }
    }
    if (!me.live) return;
    float* to = k.part + row * (k.SB + 2) * a.C + c;
#pragma unroll
    for (int s = 0; s < SP; s++) to[(int64_t)(me.s0 + s) * a.C] = dA[s];
    if (slice == 0) {
        to[(int64_t)k.SB * a.C] = dD;
        to[(int64_t)(k.SB + 1) * a.C] = dbias;
    }
}

// dB and dC from the rows that the workgroups of a group's channels left.
template <class T> __global__ void __launch_bounds__(256) k_scan_join(Scan k) {
    const MoScan& a = k.a;
    const int64_t rows = a.T * a.N * a.G, id = block_here() * 256 + threadIdx.x, row = id / (2 * k.SB);
    if (row >= rows) return;
    const int i = (int)(id % (2 * k.SB)), s = i % k.SB, g = (int)(row % a.G);
    if (s >= a.S) return;
    float x = 0.f;
    for (int p = 0; p < k.cuts; p++) x += k.part_bc[p * rows * 2 * k.SB + id];
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
        if (k.segments > 1) {
            dim3 grid, block;
            scan_launch_shape(k, k.segments * a.N * a.G * k.per, grid, block);
            hipLaunchKernelGGL((k_scan_back_sums<T, SP, SPLIT>), grid, block, 0, s, k);
            hipLaunchKernelGGL((k_scan_enter<true>), grid_of((a.N * k.SB * a.C + 255) / 256), dim3(256), 0, s, k);
        }
        const int waves = k.across * k.slices;
        hipLaunchKernelGGL((k_scan_back<T, SP, SPLIT>), grid_of(k.rows * a.G * k.cuts), dim3(kWave * waves), waves * back_wave_lds<T>(), s, k);
        if (launched("k_scan_back")) return -1;
        const int64_t n = a.T * a.N * a.G * 2 * k.SB;
        if (n && k.cuts > 1) hipLaunchKernelGGL((k_scan_join<T>), grid_of((n + 255) / 256), dim3(256), 0, s, k);
        if (launched("k_scan_join")) return -1;
        if (!a.dA && !a.dD && !a.ddt_bias) return 0;
        return column_sums(ColumnSums{k.part, more, k.rows, k.SB + 2, a.C, a.S, k.SB, a.dA, a.dD, a.ddt_bias}, s);
    });
}

}  // namespace mo
