// The gradient of the selective state space scan.
#pragma once
#include "scan.hpp"

namespace mo {

// Back through the chunks from the states kept before each: a chunk's states are made again and stay in registers, then the steps go
// backwards with Q, the gradient of the state after a step from all later ones:
//   R = C dy + Q,  dC = sum_c h dy,  dB = sum_c R u,  du = sum_s R B,  Q = R a,  q = Q h_{t-1},  dA += q d,  dd = du x + sum_s q A
// (u = d x, a = exp(d A); Q and q are 0 where the episode starts). The sums over channels are joined in the wave (wave_sums), then in LDS over the
// workgroup's waves, which have neighbouring channels of one env and segment.
// The 8 x 16 states of a chunk take half of a wave's 256 registers, so two waves share a SIMD; the other way round, states kept for every step would be
// 64 bytes a channel to write and read where all else is 22. Bound by the vector units and by two waves' waits: 128 steps x 2,048 envs x
// 512 channels of 16 states in bf16 2,210 us, the units busy 72 % of them with 400 instructions a step (half of it the states again and the sums over
// lanes). One wave a SIMD with spills in the steps took 6,400; steps that wait for their own inputs 4,240; sums over lanes by swaps
// alone 2,570.
constexpr int BACK_WAVES = SCAN_BACK_WAVES;

// Where bit I of cuts is set: x = y = 0, for all states.
template <int I> __device__ __forceinline__ void if_start_clear8(unsigned cuts, float* x, float* y) {
    asm volatile(
        "s_bitcmp1_b32 %[m], %[i]\n\ts_cbranch_scc0 .Lstart%=\n\t"
        "v_mov_b32 %0, 0\n\tv_mov_b32 %1, 0\n\tv_mov_b32 %2, 0\n\tv_mov_b32 %3, 0\n\tv_mov_b32 %4, 0\n\tv_mov_b32 %5, 0\n\tv_mov_b32 %6, 0\n\tv_mov_b32 %7, 0\n\t"
        "v_mov_b32 %8, 0\n\tv_mov_b32 %9, 0\n\tv_mov_b32 %10, 0\n\tv_mov_b32 %11, 0\n\tv_mov_b32 %12, 0\n\tv_mov_b32 %13, 0\n\tv_mov_b32 %14, 0\n\tv_mov_b32 %15, 0\n"
        ".Lstart%=:"
        : "+v"(x[0]), "+v"(x[1]), "+v"(x[2]), "+v"(x[3]), "+v"(x[4]), "+v"(x[5]), "+v"(x[6]), "+v"(x[7]),
          "+v"(y[0]), "+v"(y[1]), "+v"(y[2]), "+v"(y[3]), "+v"(y[4]), "+v"(y[5]), "+v"(y[6]), "+v"(y[7])
        : [m] "s"(cuts), [i] "n"(I)
        : "scc");
}
template <int I> __device__ __forceinline__ void if_start_clear4(unsigned cuts, float* x, float* y) {
    asm volatile(
        "s_bitcmp1_b32 %[m], %[i]\n\ts_cbranch_scc0 .Lstart%=\n\tv_mov_b32 %0, 0\n\tv_mov_b32 %1, 0\n\tv_mov_b32 %2, 0\n\tv_mov_b32 %3, 0\n\t"
        "v_mov_b32 %4, 0\n\tv_mov_b32 %5, 0\n\tv_mov_b32 %6, 0\n\tv_mov_b32 %7, 0\n.Lstart%=:"
        : "+v"(x[0]), "+v"(x[1]), "+v"(x[2]), "+v"(x[3]), "+v"(y[0]), "+v"(y[1]), "+v"(y[2]), "+v"(y[3])
        : [m] "s"(cuts), [i] "n"(I)
        : "scc");
}
template <int I, int SP> __device__ __forceinline__ void if_start_clear(unsigned cuts, float (&x)[SP], float (&y)[SP]) {
#pragma unroll
    for (int s = 0; s < SP / 8 * 8; s += 8) if_start_clear8<I>(cuts, x + s, y + s);
    if constexpr (SP % 8 == 4) if_start_clear4<I>(cuts, x + SP - 4, y + SP - 4);
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

// Workgroups of `across` waves of channels by `slices`. A wave's own LDS: the tiles of x, dt, z and dout (whose places dx, ddt and dz take); of each step
// its size d, d's slope by dt, dy and y; the sums for its workgroup's dB and dC (of two chunks in turn, but where a second barrier follows); dA up to the last chunk; where waves share
// channels, du and dd. With float32 tiles dy takes dout's place, what dz has of dout and z takes z's, and dd takes dt's.
template <class T, int SP, bool SPLIT> struct BackLds {
    static constexpr int TILE = SCAN_STEPS * kWave, TURN = SCAN_STEPS * 32, SUMS = (SPLIT ? 1 : 2) * TURN;
    static constexpr bool F32 = sizeof(T) == 4;
    static constexpr int BYTES = scan_back_lds(sizeof(T), SP, SPLIT);
    T* t;
    __device__ __forceinline__ explicit BackLds(char* p) : t((T*)p) {}
    __device__ __forceinline__ T* x() const { return t; }
    __device__ __forceinline__ T* dt() const { return t + TILE; }
    __device__ __forceinline__ T* z() const { return t + 2 * TILE; }
    __device__ __forceinline__ T* dout() const { return t + 3 * TILE; }
    __device__ __forceinline__ float* d() const { return (float*)(t + 4 * TILE); }
    __device__ __forceinline__ float* slope() const { return d() + TILE; }
    __device__ __forceinline__ float* y() const { return d() + 2 * TILE; }
    __device__ __forceinline__ float* sums(int64_t chunk) const { return d() + 3 * TILE + (SPLIT ? 0 : (chunk & 1) * TURN); }   // (SCAN_STEPS, 32)
    __device__ __forceinline__ float* dA() const { return d() + 3 * TILE + SUMS; }           // (SP, lanes)
    __device__ __forceinline__ float* dy() const { return F32 ? (float*)dout() : dA() + SP * kWave; }
    __device__ __forceinline__ float* du() const { return dA() + SP * kWave + (F32 ? 0 : TILE); }
    __device__ __forceinline__ float* dd() const { return F32 ? (float*)dt() : du() + TILE; }
};
// The part of dz that the step's y does not change.
__device__ __forceinline__ float gate_slope(float dout, float z, float sig) { return dout * (sig * fmaf(z, 1.f - sig, 1.f)); }
// sum + x, and what its rounding takes in `rest`, for the next one (compensated summation).
__device__ __forceinline__ void add_to(float& sum, float& rest, float x) {
    const float y = x - rest, s = sum + y;
    rest = (s - sum) - y;
    sum = s;
}

template <class T, int SP, bool SPLIT, bool PAD>
__global__ void __launch_bounds__(BACK_WAVES* kWave, 2) k_scan_back(Scan k) {
    const MoScan& a = k.a;
    typedef BackLds<T, SP, SPLIT> Lds;
    extern __shared__ __attribute__((aligned(16))) char lds[];
    const int w = wave_here(), slices = SPLIT ? k.slices : 1, slice = SPLIT ? w % slices : 0, across = w / slices;
    const int64_t items = k.segments * a.N, row = block_here() / (a.G * k.cuts), bg = block_here() % (a.G * k.cuts);
    if (row >= k.rows) return;
    const int g0 = (int)(bg / k.cuts), cut = (int)(bg % k.cuts), in_group = cut * k.across + across;   // (waves past the group's channels join the barriers only)
    const int cb = g0 * k.per + min(in_group, k.per - 1);
    const Lds l(lds + w * Lds::BYTES);
    const bool gate = a.z.p;
    ScanPlace place(k, row, cb, slice, SP);
    if (in_group >= k.per) { place.live = false; place.there = 0; }
    const Real<SP, SPLIT, PAD> real(a.S - place.s0);
    float A[SP], dD = 0.f, dbias = 0.f, dD_rest = 0.f, dbias_rest = 0.f;
    const int c = place.c;
    load_decays<SP>(a, place, A);
    const float bias = a.dt_bias ? a.dt_bias[c] : 0.f, D = a.D ? a.D[c] : 0.f;
#pragma unroll
    for (int s = 0; s < SP; s++) l.dA()[s * kWave + place.lane] = 0.f;
    for (int64_t item = row; item < items; item += k.rows) {
        const int64_t n = place.n = item % a.N;
        place.segment = item / a.N;
        const int64_t first = place.segment * k.each, last = min(k.chunks, first + k.each);
        float Q[SP], before[SP], touch = 0.f, touch_h = 0.f;
        ChunkIn<T> ix, idt, iz, ido;
        uint8_t flag = 0;
        const auto ahead = [&](int64_t chunk) {
            const Scan& k = args_again();
            const ScanPlace me = place.again();
            const int lane = me.lane;
            const int64_t t0 = chunk * SCAN_STEPS;
            const int steps = (int)min((int64_t)SCAN_STEPS, k.a.T - t0);
            flag = start_of_lane(k.a, t0, steps, me);
            // (a lane for each 64 bytes of the chunk's B and C, which the scalar loads then find in the L2)
            const int64_t row = ((t0 + lane % SCAN_STEPS) * k.a.N + n) * k.a.G + g0;
            touch = k.bc[row * 2 * k.SB + min(lane / SCAN_STEPS * 16, 2 * k.SB - 1)];
            // (and one for each 128 bytes of the states before it)
            touch_h = k.kept[((chunk * k.a.N + n) * k.SB + me.s0 + min(lane / 2, SP - 1)) * k.a.C + me.c0 + min(lane % 2 * 32, max(me.there - 1, 0))];
            if (!k.wide) return;
            ix.ahead(k.a.x, t0, steps, me);
            idt.ahead(k.a.dt, t0, steps, me);
            if (gate) iz.ahead(k.a.z, t0, steps, me);
            ido.ahead(k.a.dout, t0, steps, me);
        };
        // the states before a chunk: into registers that are free between two chunks
        const auto states_ahead = [&](int64_t chunk) {
            const Scan& k = args_again();
            const ScanPlace me = place.again();
            const float* from = k.kept + ((chunk * k.a.N + n) * k.SB + me.s0) * k.a.C + me.c0;
#pragma unroll
            for (int s = 0; s < SP; s++) before[s] = __builtin_nontemporal_load(lane_at(from + (int64_t)s * k.a.C, me.at * 4));
        };
        if (first < last) {
            ahead(last - 1);
            states_ahead(last - 1);
        }
        if (k.segments == 1) load_states<SP>(a, a.dstate_out, n, c, place.s0, Q);
        else
#pragma unroll
            for (int s = 0; s < SP; s++) Q[s] = k.seg_h[((place.segment * a.N + n) * k.SB + place.s0 + s) * a.C + c];
#pragma unroll
        for (int s = 0; s < SP; s++) Q[s] = place.live ? real(Q[s], s) : 0.f;
        // what a chunk left in LDS goes to memory
        const auto after_chunk = [&](int64_t chunk, int64_t t0, int steps) {
            const Scan& k = args_again();
            const MoScan& a = k.a;
            const ScanPlace me = place.again();
            const int lane = me.lane, c = me.c;
            if constexpr (SPLIT) {
                const uint32_t with_D = mask_of(a.D);
                for (int i = slice; i < steps; i += slices) {
                    const int at = i * kWave + lane;
                    float y = 0.f, du = 0.f, dd = 0.f;
                    for (int s = 0; s < slices; s++) {
                        const Lds o(lds + (w - slice + s) * Lds::BYTES);
                        y += o.y()[at];
                        du += o.du()[at];
                        dd += o.dd()[at];
                    }
                    const float x = as_f32(l.x()[at]), dy = l.dy()[at], ddt = fmaf(du, x, dd * LN2) * l.slope()[at];
                    add_to(dD, dD_rest, dy * x);
                    add_to(dbias, dbias_rest, ddt);
                    if (!me.live) continue;
                    const auto row_of = [&](const MoRows& r) { return (T*)r.p + (t0 + i) * r.st + n * r.sn + c; };
                    *row_of(a.dx) = as<T>(fmaf(du, l.d()[at], D * masked(dy, with_D)));
                    *row_of(a.ddt) = as<T>(ddt);
                    if (!gate) continue;
                    const float z = as_f32(l.z()[at]);
                    *row_of(a.dz) = as<T>(fmaf(D, masked(x, with_D), y) * (Lds::F32 ? z : gate_slope(as_f32(l.dout()[at]), z, sigmoid(z))));
                }
            } else {
                ChunkIn<T>::leave(l.x(), a.dx, t0, steps, me, k.wide);
                ChunkIn<T>::leave(l.dt(), a.ddt, t0, steps, me, k.wide);
                if (gate) ChunkIn<T>::leave(l.z(), a.dz, t0, steps, me, k.wide);
            }
            // dB and dC of the chunk: the workgroup's waves joined (the next chunk's sums go to the other place)
            const int SB = SPLIT ? k.SB : SP;
            float* const part = k.part_bc + ((((int64_t)cut * a.T + t0) * a.N + n) * a.G + g0) * 2 * SB;
            T* const dB = (T*)a.dB.p + t0 * a.dB.st + n * a.dB.sn + g0 * a.dB.sh;
            T* const dC = (T*)a.dC.p + t0 * a.dC.st + n * a.dC.sn + g0 * a.dC.sh;
            for (int i = w * kWave + lane; i < steps * 2 * SB; i += blockDim.x) {
                const int j = i / (2 * SB), m = i % (2 * SB), which = m / SB, s = m % SB, of = s / SP;
                float x = 0.f;
                for (int v = of; v < k.across * slices; v += slices)
                    x += Lds(lds + v * Lds::BYTES).sums(chunk)[j * 32 + which * SP + s % SP];
                if (k.cuts > 1) part[j * a.N * a.G * 2 * SB + m] = x;
                else if (s < a.S) (which ? dC : dB)[j * (which ? a.dC.st : a.dB.st) + s] = as<T>(x);
            }
            if constexpr (SPLIT) __syncthreads();             // (their partial sums have been read)
        };
        for (int64_t chunk = last - 1; chunk >= first; chunk--) {
            const Scan& k = args_again();
            const MoScan& a = k.a;
            const ScanPlace me = place.again();
            const int lane = me.lane;
            const int64_t t0 = chunk * SCAN_STEPS;
            const int steps = (int)min((int64_t)SCAN_STEPS, a.T - t0);
            const unsigned cuts = (unsigned)__ballot(flag != 0);
            asm volatile("" ::"v"(touch));
            wave_wrote();
            if (k.wide) {
                ix.arrive(l.x(), steps, me);
                idt.arrive(l.dt(), steps, me, NO_SIZE<T>);
                if (gate) iz.arrive(l.z(), steps, me);
                ido.arrive(l.dout(), steps, me);
            } else {
                ChunkIn<T>::narrow(l.x(), a.x, t0, steps, me);
                ChunkIn<T>::narrow(l.dt(), a.dt, t0, steps, me, -INFINITY);
                if (gate) ChunkIn<T>::narrow(l.z(), a.z, t0, steps, me);
                ChunkIn<T>::narrow(l.dout(), a.dout, t0, steps, me);
            }
            wave_wrote();
#pragma unroll
            for (int i = 0; i < SCAN_STEPS; i++) {
                const int at = i * kWave + lane;
                const Size p = softplus(as_f32(l.dt()[at]) + bias);
                l.d()[at] = p.d;
                l.slope()[at] = p.slope;
                const float dout = as_f32(l.dout()[at]);
                if (gate) {
                    const float z = as_f32(l.z()[at]), sig = sigmoid(z);
                    if constexpr (Lds::F32) l.z()[at] = gate_slope(dout, z, sig);
                    l.dy()[at] = dout * (z * sig);
                } else if constexpr (!Lds::F32) {
                    l.dy()[at] = dout;
                }
            }
            end_of_step();
            float h[SCAN_STEPS][SP];                          // the states before each step
#pragma unroll
            for (int s = 0; s < SP; s++) h[0][s] = me.live ? before[s] : 0.f;
            float* const to_join = l.sums(chunk);
            const uint32_t with_D = mask_of(a.D);
            // what a step needs, read a step ahead
            struct In { float d, dy; T x; };
            const auto in_of = [&](int i) { return In{l.d()[i * kWave + lane], l.dy()[i * kWave + lane], l.x()[i * kWave + lane]}; };
            const int64_t bc_step = a.N * a.G * 2 * k.SB;
            const int SB = k.SB;
            Uniform bc = uniform(k.bc + ((t0 * a.N + n) * a.G + g0) * 2 * SB + me.s0);
            StepBC<SP> now;
            load_bc<SP>(now, bc, SB);
            In in = in_of(0);
            // the states again, y and dC
            each_step([&](auto step) {
                constexpr int i = decltype(step)::value;
                StepBC<SP> next;
                In in_next;
                if constexpr (i + 1 < SCAN_STEPS) {
                    bc = move_on(bc, bc_step);
                    load_bc<SP>(next, bc, SB);
                    in_next = in_of(i + 1);
                }
                const float u = in.d * as_f32(in.x);
                float v[SP], y = 0.f;
#pragma unroll
                for (int s = 0; s < SP; s++) v[s] = fmaf(exp2_raw(in.d * A[s]), h[i][s], u * now.b[s]);
                if_start_set<i, SP>(cuts, v, u, now.b);
#pragma unroll
                for (int s = 0; s < SP; s++) {
                    v[s] = real(v[s], s);
                    if constexpr (i + 1 < SCAN_STEPS) h[i + 1][s] = v[s];
                    y = fmaf(now.c[s], v[s], y);
                    v[s] *= in.dy;
                }
                l.y()[i * kWave + lane] = y;
                const float sum = wave_sums<SP>(v);
                if (sum_slot(lane, SP) < SP) to_join[i * 32 + SP + sum_slot(lane, SP)] = sum;
                if constexpr (i + 1 < SCAN_STEPS) {
                    now = next;
                    in = in_next;
                }
                end_of_step();
            });
            if constexpr (!SPLIT) {
                if (gate)
#pragma unroll
                    for (int i = 0; i < SCAN_STEPS; i++) {
                        const int at = i * kWave + lane;
                        const float z = as_f32(l.z()[at]);
                        l.z()[at] = as<T>(fmaf(D, masked(as_f32(l.x()[at]), with_D), l.y()[at]) * (Lds::F32 ? z : gate_slope(as_f32(l.dout()[at]), z, sigmoid(z))));
                    }
                end_of_step();
            }
            // and back
            float dA[SP], dD_here = 0.f, dbias_here = 0.f;    // the chunk's own (the sum of all of them goes on in LDS)
#pragma unroll
            for (int s = 0; s < SP; s++) dA[s] = 0.f;
            load_bc<SP>(now, bc, SB);
            in = in_of(SCAN_STEPS - 1);
            each_step([&](auto step) {
                constexpr int i = SCAN_STEPS - 1 - decltype(step)::value;
                const int at = i * kWave + lane;
                StepBC<SP> next;
                In in_next;
                if constexpr (i > 0) {
                    bc = move_on(bc, -bc_step);
                    load_bc<SP>(next, bc, SB);
                    in_next = in_of(i - 1);
                }
                const float x = as_f32(in.x), u = in.d * x;
                float du = 0.f, dd = 0.f, v[SP];
#pragma unroll
                for (int s = 0; s < SP; s++) {
                    Q[s] = real(fmaf(now.c[s], in.dy, Q[s]), s);
                    du = fmaf(Q[s], now.b[s], du);
                    v[s] = Q[s] * u;
                }
                const float sum = wave_sums<SP>(v);
                if (sum_slot(lane, SP) < SP) to_join[i * 32 + sum_slot(lane, SP)] = sum;
                made(du);
                end_of_step();
#pragma unroll
                for (int s = 0; s < SP; s++) {
                    Q[s] *= exp2_raw(in.d * A[s]);
                    v[s] = Q[s] * h[i][s];
                }
                if_start_clear<i, SP>(cuts, Q, v);
#pragma unroll
                for (int s = 0; s < SP; s++) {
                    dd = fmaf(v[s], A[s], dd);
                    dA[s] = fmaf(v[s], in.d, dA[s]);
                }
                if constexpr (SPLIT) {
                    l.du()[at] = du;
                    l.dd()[at] = dd;
                } else {
                    const float ddt = fmaf(du, x, dd * LN2) * l.slope()[at];
                    dD_here = fmaf(in.dy, x, dD_here);
                    dbias_here += ddt;
                    l.x()[at] = as<T>(fmaf(du, in.d, D * masked(in.dy, with_D)));
                    l.dt()[at] = as<T>(ddt);
                }
                if constexpr (i > 0) {
                    now = next;
                    in = in_next;
                }
                if constexpr (i == SCAN_STEPS / 2) {
                    if (chunk > first) ahead(chunk - 1);      // (the states that are done with have left their registers)
                }
                end_of_step();
            });
#pragma unroll
            for (int s = 0; s < SP; s++) l.dA()[s * kWave + lane] += dA[s];
            if constexpr (!SPLIT) {
                add_to(dD, dD_rest, dD_here);
                add_to(dbias, dbias_rest, dbias_here);
            }
            if (chunk > first) {
                asm volatile("" ::"v"(touch_h));
                states_ahead(chunk - 1);
            }
            __syncthreads();
            after_chunk(chunk, t0, steps);
        }
        if (first == 0 && a.dstate && place.live) store_states<SP>(a, a.dstate, n, c, place.s0, Q);
        __syncthreads();                                      // (one env's last sums are read before the next one's first)
    }
    const ScanPlace& me = place;
    const int lane = me.lane;
    if constexpr (SPLIT) {
        l.du()[lane] = dD;
        l.dd()[lane] = dbias;
        __syncthreads();
        dD = dbias = 0.f;
        for (int s = 0; s < slices; s++) {
            const Lds o(lds + (w - slice + s) * Lds::BYTES);
            dD += o.du()[lane];
            dbias += o.dd()[lane];
        }
    }
    if (!me.live) return;
    float* to = k.part + row * (k.SB + 2) * a.C + c;
#pragma unroll
    for (int s = 0; s < SP; s++) to[(int64_t)(me.s0 + s) * a.C] = l.dA()[s * kWave + lane];
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
    return by_states(k, [&](auto sp, auto split, auto pad) {
        constexpr int SP = decltype(sp)::value;
        constexpr bool SPLIT = decltype(split)::value, PAD = decltype(pad)::value;
        if (k.segments > 1) {
            dim3 grid, block;
            scan_launch_shape(k, k.segments * a.N * a.G * k.per, grid, block);
            hipLaunchKernelGGL((k_scan_back_sums<T, SP, SPLIT>), grid, block, 0, s, k);
            hipLaunchKernelGGL((k_scan_enter<true>), grid_of((a.N * k.SB * a.C + 255) / 256), dim3(256), 0, s, k);
        }
        const int waves = k.across * k.slices;
        static_assert(scan_back_lds(sizeof(T), 16, false) * SCAN_BACK_WAVES <= 160 << 10, "");
        hipLaunchKernelGGL((k_scan_back<T, SP, SPLIT, PAD>), grid_of(k.rows * a.G * k.cuts), dim3(kWave * waves), waves * (BackLds<T, SP, SPLIT>::BYTES), s, k);
        if (launched("k_scan_back")) return -1;
        const int64_t n = a.T * a.N * a.G * 2 * k.SB;
        if (n && k.cuts > 1) hipLaunchKernelGGL((k_scan_join<T>), grid_of((n + 255) / 256), dim3(256), 0, s, k);
        if (launched("k_scan_join")) return -1;
        if (!a.dA && !a.dD && !a.ddt_bias) return 0;
        return column_sums(ColumnSums{k.part, more, k.rows, k.SB + 2, a.C, a.S, k.SB, a.dA, a.dD, a.ddt_bias}, s);
    });
}

}  // namespace mo
