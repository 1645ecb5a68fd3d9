// The selective state space scan over the steps of a rollout.
#pragma once
#include <utility>

#include "sums.hpp"

namespace mo {

// A wave has 64 channels of one env, a lane all of a channel's states (or SP of them: then up to four waves share the channels and join their
// sums in LDS). B and C are the same for all lanes: they lie packed in float32 (k_scan_pack) and come as scalar loads a step ahead, so a step of a
// state is one exponential, two products and two fused multiply-adds on registers. x, dt and z come in 16-byte pieces of whole rows, a
// chunk of steps ahead, and go to their lanes through LDS; results leave the same way.
// Bound by the vector units: 24 cycles a state and wave (an exponential takes 8 of them), about 130 more a step for sizes, gates and rounding. 128
// steps x 2,048 envs x 512 channels of 16 states in bf16, the states for the gradient kept: 570 us, the units busy all the time (they make
// 3.8e12 states a second; memory moves 2.3 GB meanwhile). With rows an element a lane, B and C all steps at once and their registers spilled: 1,087.
constexpr int SCAN_STEPS = 8;        // steps of a chunk: between two kept states
constexpr int SCAN_WAVES = 4;
constexpr float LOG2E = 1.44269504088896340736f, LN2 = 0.69314718055994530942f;

struct Scan {
    MoScan a;
    const float* bc;                 // (whole chunks of steps and a step more, N, G, 2, SB): B and C padded with zeros to whole slices
    float* kept;                     // (chunks, N, SB, C): the states before each chunk, for the gradient; or null
    float *seg_h, *seg_d;            // (segments, N, SB, C), (segments, N, C): see k_scan_enter
    float *part_bc, *part;           // (gradient) (cuts, T, N, G, 2, SB), (rows, SB + 2, C)
    int64_t chunks, each, segments;  // chunks of all steps, and of a segment
    int64_t rows;                    // (gradient) envs' segments that are taken at a time
    int slices, SB, Cg, per;         // waves that share channels, states padded, channels of a group, waves that span them
    int across, cuts;                // (gradient) waves of channels a workgroup, workgroups of a group's channels
    int wide;                        // all rows of channels lie on 16 bytes, in whole pieces
};

typedef const float __attribute__((address_space(4))) * Uniform;   // read by scalar loads: the same for all lanes, not written meanwhile
__device__ __forceinline__ Uniform uniform(const float* p) { return (Uniform)(uintptr_t)p; }

__device__ __forceinline__ float exp2_raw(float x) { return __builtin_amdgcn_exp2f(x); }
// softplus(r) = max(r, 0) + log1p(e), e = exp(-|r|) <= 1. With t = 1 + e rounded, log1p(e) = log(t) + (e - (t - 1)): the instruction's logarithm is
// within 2^-23 of its value down to t = 1, and what the rounding of t took is added (its own derivative 1 / t left out is 2^-25 e at most).
struct Size { float d, slope; };     // and its derivative, 1 / (1 + exp(-r))
__device__ __forceinline__ Size softplus(float r) {
    const float e = exp2_raw(-fabsf(r) * LOG2E), t = 1.f + e, rest = e - (t - 1.f);
    return {fmaxf(r, 0.f) + fmaf(__builtin_amdgcn_logf(t), LN2, rest), (r < 0.f ? e : 1.f) * __builtin_amdgcn_rcpf(t)};
}
__device__ __forceinline__ float sigmoid(float z) { return __builtin_amdgcn_rcpf(1.f + exp2_raw(-z * LOG2E)); }

// B and C of every step in float32, padded.
__host__ __device__ __forceinline__ int64_t scan_rows(const Scan& k) { return k.chunks * SCAN_STEPS + 1; }
template <class T> __global__ void __launch_bounds__(256) k_scan_pack(Scan k, float* bc) {   // (four values a thread: fewer workgroups to start)
    const MoScan& a = k.a;
    const int64_t id = block_here() * 256 + threadIdx.x, row = id / (k.SB / 2);
    const int i = (int)(id % (k.SB / 2)) * 4, s = i % k.SB, g = (int)(row % a.G);
    const int64_t n = row / a.G % a.N, t = row / a.G / a.N;
    if (t >= scan_rows(k)) return;
    const MoRows& r = i < k.SB ? a.Bt : a.Ct;
    const T* from = (const T*)r.p + t * r.st + n * r.sn + g * r.sh + s;
    Pack<float, 4> x{};
    if (t < a.T)
#pragma unroll
        for (int j = 0; j < 4; j++)
            if (s + j < a.S) x.v[j] = as_f32(from[j]);
    *(Pack<float, 4>*)(bc + 4 * id) = x;
}

// All ones or none, in a scalar register; and x, or 0 whatever x is (0 times an infinity is none). One instruction with a scalar operand: the compiler would
// make a select of it, whose masks take two registers each.
__device__ __forceinline__ uint32_t mask_of(bool there) {
    uint32_t m = __builtin_amdgcn_readfirstlane(there ? -1 : 0);
    asm("" : "+s"(m));
    return m;
}
__device__ __forceinline__ float masked(float x, uint32_t m) { return __uint_as_float(__float_as_uint(x) & m); }

// Where a lane has registers for more states than there are (PAD), the rest stay 0: a product of 0 and an infinite d x would not be, and so
// reach y and the gradients of step sizes. Without slices at most three of a lane's states are not there, in the last slice most may not be. Kernels of
// their own, for the masks take an instruction for each such state and step (128 x 512 x 512, bf16, forward and gradient, without and with them: 13
// states 748 and 801 us, 20 states 1,255 and 1,331, 49 states 3,771 and 4,029).
template <int SP, bool SPLIT, bool PAD> struct Real {
    static constexpr int FROM = !PAD ? SP : SPLIT ? 0 : SP - 3;   // those before are there
    uint32_t m[PAD ? SP - FROM : 1];
    __device__ __forceinline__ explicit Real(int there) {
#pragma unroll
        for (int s = FROM; s < SP; s++) m[s - FROM] = mask_of(s < there);
    }
    __device__ __forceinline__ float operator()(float x, int s) const { return s < FROM ? x : masked(x, m[s < FROM ? 0 : s - FROM]); }
};

// What a wave works on.
struct ScanPlace {
    int64_t n, segment;
    int g, c0, c, lane, s0, there;   // group, first channel, this lane's, its first state, channels that there are
    uint32_t at;                     // this lane's channel, from the first (the last one that there is, where there are fewer)
    bool live;
    __device__ __forceinline__ ScanPlace(const Scan& k, int64_t item, int cb, int slice, int SP) {
        n = item % k.a.N;
        segment = item / k.a.N;
        g = cb / k.per;
        lane = threadIdx.x % kWave;
        const int i = cb % k.per * kWave;
        there = min(kWave, k.Cg - i);
        live = lane < there;
        c0 = g * k.Cg + i;
        at = min(lane, there - 1);
        c = c0 + (int)at;
        s0 = slice * SP;
    }
    // The same, the lane's own values made anew from here on: they would be kept through the steps.
    __device__ __forceinline__ ScanPlace again() const {
        ScanPlace p = *this;
        asm volatile("" : "+v"(p.lane));
        p.live = p.lane < there;
        p.at = max(0, min(p.lane, there - 1));
        p.c = c0 + (int)p.at;
        return p;
    }
};
__device__ __forceinline__ int wave_here() { return __builtin_amdgcn_readfirstlane(threadIdx.x / kWave); }
// The wave's own LDS: what its lanes wrote is there for its other lanes.
__device__ __forceinline__ void wave_wrote() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// The kernel's arguments, read again from here on: kept in registers through the steps they would push the steps' own out.
__device__ __forceinline__ const Scan& args_again() {
    typedef const Scan __attribute__((address_space(4))) * Args;
    uint64_t p = (uint64_t)__builtin_amdgcn_kernarg_segment_ptr();
    asm volatile("" : "+s"(p));
    return *(const Scan*)(Args)p;
}
// A lane's place behind a pointer that all lanes share: a 32-bit offset, so that the pointer stays in scalar registers.
template <class P> __device__ __forceinline__ P* lane_at(P* p, uint32_t bytes) {
    return (P*)((std::conditional_t<std::is_const_v<P>, const char, char>*)p + bytes);
}
// A chunk's rows of 64 channels, zeros where there are none (rows past the last step, channels past the group's). Wide: in 16-byte pieces through
// registers (ahead of their use); else an element a lane. Where there are none, a place that there is is read and not used: no branches.
template <class T> struct ChunkIn {
    static constexpr int EPV = 16 / sizeof(T), PR = kWave / EPV, ROWS = kWave / PR, N = SCAN_STEPS / ROWS;
    uint4 v[N];
    static __device__ __forceinline__ T* base(const MoRows& r, int64_t t0, const ScanPlace& me) { return (T*)r.p + t0 * r.st + me.n * r.sn + me.c0; }
    static __device__ __forceinline__ uint32_t piece(const MoRows& r, const ScanPlace& me, int row) {   // (a chunk spans less than 2^31 bytes)
        const int p = me.lane % PR * EPV;
        return ((uint32_t)row * (uint32_t)r.st + (p < me.there ? p : 0)) * (uint32_t)sizeof(T);
    }
    __device__ __forceinline__ void ahead(const MoRows& r, int64_t t0, int steps, const ScanPlace& me) {
#pragma unroll
        for (int i = 0; i < N; i++) v[i] = *(const uint4*)lane_at((const T*)base(r, t0, me), piece(r, me, min(me.lane / PR + i * ROWS, steps - 1)));
    }
    __device__ __forceinline__ void arrive(T* to, int steps, const ScanPlace& me, uint32_t none = 0) const {
#pragma unroll
        for (int i = 0; i < N; i++) {
            const bool there = me.lane / PR + i * ROWS < steps && me.lane % PR * EPV < me.there;
            *(uint4*)(to + (i * kWave + me.lane) * EPV) = there ? v[i] : uint4{none, none, none, none};
        }
    }
    static __device__ __forceinline__ void narrow(T* to, const MoRows& r, int64_t t0, int steps, const ScanPlace& me, float none = 0.f) {
        const T* p = base(r, t0, me);
        T x[SCAN_STEPS];
#pragma unroll
        for (int i = 0; i < SCAN_STEPS; i++) {
            x[i] = *lane_at(p, me.at * (uint32_t)sizeof(T));
            if (i + 1 < steps) p += r.st;
        }
#pragma unroll
        for (int i = 0; i < SCAN_STEPS; i++) to[i * kWave + me.lane] = me.live && i < steps ? x[i] : as<T>(none);
    }
    // the other way, from LDS to memory
    static __device__ __forceinline__ void leave(const T* from, const MoRows& r, int64_t t0, int steps, const ScanPlace& me, bool wide) {
        if (wide) {
#pragma unroll
            for (int i = 0; i < N; i++)
                if (me.lane / PR + i * ROWS < steps && me.lane % PR * EPV < me.there)
                    stream((uint4*)lane_at(base(r, t0, me), piece(r, me, me.lane / PR + i * ROWS)), *(const uint4*)(from + (i * kWave + me.lane) * EPV));
        } else if (me.live) {
            T* p = base(r, t0, me);
            for (int i = 0; i < steps; i++, p += r.st) *lane_at(p, me.at * (uint32_t)sizeof(T)) = from[i * kWave + me.lane];
        }
    }
};
// In the place of a dt that is not there: minus infinity, a step of no size, which changes nothing.
template <class T> constexpr uint32_t NO_SIZE = 0xff800000u;
template <> inline constexpr uint32_t NO_SIZE<bf16> = 0xff80ff80u;
// Which of the SCAN_STEPS steps from t0 start an episode: lane i has step i's flag.
__device__ __forceinline__ uint8_t start_of_lane(const MoScan& a, int64_t t0, int steps, const ScanPlace& me) {
    return a.start && me.lane < steps ? a.start[(t0 + me.lane) * a.N + me.n] : 0;
}
template <int SP> __device__ __forceinline__ void load_decays(const MoScan& a, const ScanPlace& me, float (&A)[SP]) {
#pragma unroll
    for (int s = 0; s < SP; s++) A[s] = !me.live ? 0.f : me.s0 + s < a.S ? a.A[(int64_t)me.c * a.S + me.s0 + s] * LOG2E : -1.f;   // (0 times an infinite d is none)
}
// A channel's states as they lie, zeros past the last (or of none); in 16-byte accesses where they allow it (a lane's states lie 4 S
// bytes from its neighbour's).
__device__ __forceinline__ bool in_fours(const MoScan& a, const float* p) { return a.S % 4 == 0 && (uintptr_t)p % 16 == 0; }
template <int SP> __device__ __forceinline__ void load_states(const MoScan& a, const float* p, int64_t n, int c, int s0, float (&h)[SP]) {
    const float* from = p + (n * a.C + c) * a.S + s0;
    if (p && in_fours(a, p)) {
#pragma unroll
        for (int s = 0; s < SP; s += 4) *(Pack<float, 4>*)(h + s) = s0 + s < a.S ? *(const Pack<float, 4>*)(from + s) : Pack<float, 4>{};
    } else {
#pragma unroll
        for (int s = 0; s < SP; s++) h[s] = p && s0 + s < a.S ? from[s] : 0.f;
    }
}
template <int SP> __device__ __forceinline__ void store_states(const MoScan& a, float* p, int64_t n, int c, int s0, const float (&h)[SP]) {
    float* to = p + (n * a.C + c) * a.S + s0;
    if (in_fours(a, p)) {
#pragma unroll
        for (int s = 0; s < SP; s += 4)
            if (s0 + s < a.S) *(Pack<float, 4>*)(to + s) = *(const Pack<float, 4>*)(h + s);
    } else {
#pragma unroll
        for (int s = 0; s < SP; s++)
            if (s0 + s < a.S) to[s] = h[s];
    }
}
// A step's B and C, in scalar registers. Loaded a step ahead; nothing moves over the end of a step, or all steps' loads would come first and
// take more registers than there are.
template <int SP> struct StepBC { float b[SP], c[SP]; };
template <int SP, bool WITH_C = true> __device__ __forceinline__ void load_bc(StepBC<SP>& v, Uniform p, int SB) {
#pragma unroll
    for (int s = 0; s < SP; s++) {
        v.b[s] = p[s];
        if (WITH_C) v.c[s] = p[SB + s];
    }
}
// Where bit I of cuts is set: h = u b, for all states. A branch of the whole wave that the compiler does not see: the steps stay one block.
template <int I> __device__ __forceinline__ void if_start_set8(unsigned cuts, float* h, float u, const float* b) {
    asm volatile(
        "s_bitcmp1_b32 %[m], %[i]\n\ts_cbranch_scc0 .Lstart%=\n\t"
        "v_mul_f32 %0, %[u], %8\n\tv_mul_f32 %1, %[u], %9\n\tv_mul_f32 %2, %[u], %10\n\tv_mul_f32 %3, %[u], %11\n\t"
        "v_mul_f32 %4, %[u], %12\n\tv_mul_f32 %5, %[u], %13\n\tv_mul_f32 %6, %[u], %14\n\tv_mul_f32 %7, %[u], %15\n.Lstart%=:"
        : "+&v"(h[0]), "+&v"(h[1]), "+&v"(h[2]), "+&v"(h[3]), "+&v"(h[4]), "+&v"(h[5]), "+&v"(h[6]), "+&v"(h[7])
        : "s"(b[0]), "s"(b[1]), "s"(b[2]), "s"(b[3]), "s"(b[4]), "s"(b[5]), "s"(b[6]), "s"(b[7]), [u] "v"(u), [m] "s"(cuts), [i] "n"(I)
        : "scc");
}
template <int I> __device__ __forceinline__ void if_start_set4(unsigned cuts, float* h, float u, const float* b) {
    asm volatile(
        "s_bitcmp1_b32 %[m], %[i]\n\ts_cbranch_scc0 .Lstart%=\n\t"
        "v_mul_f32 %0, %[u], %4\n\tv_mul_f32 %1, %[u], %5\n\tv_mul_f32 %2, %[u], %6\n\tv_mul_f32 %3, %[u], %7\n.Lstart%=:"
        : "+&v"(h[0]), "+&v"(h[1]), "+&v"(h[2]), "+&v"(h[3])
        : "s"(b[0]), "s"(b[1]), "s"(b[2]), "s"(b[3]), [u] "v"(u), [m] "s"(cuts), [i] "n"(I)
        : "scc");
}
template <int I, int SP> __device__ __forceinline__ void if_start_set(unsigned cuts, float (&h)[SP], float u, const float (&b)[SP]) {
#pragma unroll
    for (int s = 0; s < SP / 8 * 8; s += 8) if_start_set8<I>(cuts, h + s, u, b + s);
    if constexpr (SP % 8 == 4) if_start_set4<I>(cuts, h + SP - 4, u, b + SP - 4);
}
template <class F, int... I> __device__ __forceinline__ void each_step_of(F f, std::integer_sequence<int, I...>) { (f(std::integral_constant<int, I>{}), ...); }
template <class F> __device__ __forceinline__ void each_step(F f) { each_step_of(f, std::make_integer_sequence<int, SCAN_STEPS>{}); }
// p + by, known only from here on: the loads behind it come no earlier.
__device__ __forceinline__ Uniform move_on(Uniform p, int64_t by) {
    uint64_t q = (uint64_t)(p + by);
    asm volatile("" : "+s"(q));
    return (Uniform)q;
}
// What a step made is made here, not where it is used.
__device__ __forceinline__ void made(float& x) { asm volatile("" : "+v"(x)); }
__device__ __forceinline__ void end_of_step() { __builtin_amdgcn_sched_barrier(0); }

// Forward. SUMS: only what a segment adds to an entering state: its last states from zero, and the sum of its step sizes (-1 where an episode
// starts in it: nothing of what enters is left).
template <class T, int SP, bool SPLIT, bool SUMS, bool PAD>
__global__ void __launch_bounds__(SCAN_WAVES* kWave) k_scan(Scan k) {
    const MoScan& a = k.a;
    constexpr int TILE = SCAN_STEPS * kWave;
    __shared__ __attribute__((aligned(16))) T tiles[SCAN_WAVES][SUMS ? 2 : 3][TILE];
    __shared__ float part[SPLIT && !SUMS ? SCAN_WAVES : 1][SCAN_STEPS][kWave];
    const int w = wave_here(), slice = SPLIT ? w : 0, cbs = a.G * k.per;
    const int64_t wave = SPLIT ? block_here() : block_here() * SCAN_WAVES + w;
    if (wave >= k.segments * a.N * cbs) return;
    const ScanPlace place(k, wave / cbs, (int)(wave % cbs), slice, SP);
    const int64_t n = place.n, first = place.segment * k.each, last = min(k.chunks, first + k.each);
    const int c = place.c;
    T *lx = tiles[w][0], *ldt = tiles[w][1], *lz = tiles[w][SUMS ? 0 : 2];
    const bool gate = !SUMS && a.z.p;
    const Real<SP, SPLIT, PAD> real(a.S - place.s0);
    float A[SP], h[SP], total = 0.f;
    load_decays<SP>(a, place, A);
    const int64_t seg0 = ((place.segment * a.N + n) * k.SB + place.s0) * a.C + c;
    if (!SUMS && k.segments == 1) load_states<SP>(a, a.state, n, c, place.s0, h);
    else
#pragma unroll
        for (int s = 0; s < SP; s++) h[s] = SUMS ? 0.f : real(k.seg_h[seg0 + (int64_t)s * a.C], s);
    const float bias = a.dt_bias ? a.dt_bias[c] : 0.f, D = a.D ? a.D[c] : 0.f;
    ChunkIn<T> ix, idt, iz;
    uint8_t flag = 0;
    float touch = 0.f;
    const auto ahead = [&](int64_t chunk) {
        const Scan& k = args_again();
        const ScanPlace me = place.again();
        const int64_t t0 = chunk * SCAN_STEPS;
        const int steps = (int)min((int64_t)SCAN_STEPS, k.a.T - t0);
        flag = start_of_lane(k.a, t0, steps, me);
        // (a lane for each 64 bytes of the chunk's B and C, which the scalar loads then find in the L2)
        const int64_t row = ((t0 + me.lane % SCAN_STEPS) * k.a.N + n) * k.a.G + me.g;
        touch = k.bc[row * 2 * k.SB + min(me.lane / SCAN_STEPS * 16, 2 * k.SB - 1)];
        if (!k.wide) return;
        ix.ahead(k.a.x, t0, steps, me);
        idt.ahead(k.a.dt, t0, steps, me);
        if (gate) iz.ahead(k.a.z, t0, steps, me);
    };
    if (first < last) ahead(first);
    const int64_t bc_step = a.N * a.G * 2 * k.SB;
    const int SB = k.SB;
    Uniform bc = uniform(k.bc + ((first * SCAN_STEPS * a.N + n) * a.G + place.g) * 2 * SB + place.s0);
    StepBC<SP> now;
    if (first < last) load_bc<SP, !SUMS>(now, bc, SB);
    for (int64_t chunk = first; chunk < last; chunk++) {
        const Scan& k = args_again();
        const MoScan& a = k.a;
        const ScanPlace me = place.again();
        const int lane = me.lane;
        const int64_t t0 = chunk * SCAN_STEPS;
        const int steps = (int)min((int64_t)SCAN_STEPS, a.T - t0);
        const unsigned cuts = (unsigned)__ballot(flag != 0);
        asm volatile("" ::"v"(touch));
        wave_wrote();                                         // (the last chunk's results have been read)
        if (k.wide) {
            ix.arrive(lx, steps, me);
            idt.arrive(ldt, steps, me, NO_SIZE<T>);
            if (gate) iz.arrive(lz, steps, me);
        } else {
            ChunkIn<T>::narrow(lx, a.x, t0, steps, me);
            ChunkIn<T>::narrow(ldt, a.dt, t0, steps, me, -INFINITY);
            if (gate) ChunkIn<T>::narrow(lz, a.z, t0, steps, me);
        }
        wave_wrote();
        if (chunk + 1 < last) ahead(chunk + 1);
        if (!SUMS && k.kept && me.live) {
            float* to = k.kept + ((chunk * a.N + n) * k.SB + me.s0) * a.C + me.c0;
#pragma unroll
            for (int s = 0; s < SP; s++) __builtin_nontemporal_store(h[s], lane_at(to + (int64_t)s * a.C, me.at * 4));
        }
        // Nothing but the scalar loads of B and C is waited for between the steps.
        float d[SCAN_STEPS], u[SCAN_STEPS];
#pragma unroll
        for (int i = 0; i < SCAN_STEPS; i++) {
            d[i] = softplus(as_f32(ldt[i * kWave + lane]) + bias).d;
            u[i] = d[i] * as_f32(lx[i * kWave + lane]);
        }
        end_of_step();
        each_step([&](auto step) {
            constexpr int i = decltype(step)::value;
            StepBC<SP> next;
            bc = move_on(bc, bc_step);
            load_bc<SP, !SUMS>(next, bc, SB);
            float y = 0.f;
#pragma unroll
            for (int s = 0; s < SP; s++) h[s] = fmaf(exp2_raw(d[i] * A[s]), h[s], u[i] * now.b[s]);
            if_start_set<i, SP>(cuts, h, u[i], now.b);
            if (PAD)
#pragma unroll
                for (int s = 0; s < SP; s++) h[s] = real(h[s], s);
            if (!SUMS)
#pragma unroll
                for (int s = 0; s < SP; s++) y = fmaf(now.c[s], h[s], y);
            u[i] = y;
            now = next;
            made(u[i]);
            end_of_step();
        });
        if (SUMS) {
#pragma unroll
            for (int i = 0; i < SCAN_STEPS; i++) total = cuts >> i & 1 || total < 0.f ? -1.f : total + d[i];
            continue;
        }
        const uint32_t with_D = mask_of(a.D);
        const auto finish = [&](int i, float y) {
            y = fmaf(D, masked(as_f32(lx[i * kWave + lane]), with_D), y);
            if (gate) {
                const float z = as_f32(lz[i * kWave + lane]);
                y *= z * sigmoid(z);
            }
            lx[i * kWave + lane] = as<T>(y);
        };
        if (SPLIT) {                                          // (a wave finishes every `slices`th step, in its own tile)
#pragma unroll
            for (int i = 0; i < SCAN_STEPS; i++) part[slice][i][lane] = u[i];
            __syncthreads();
            for (int i = slice; i < steps; i += k.slices) {
                float y = 0.f;
                for (int s = 0; s < k.slices; s++) y += part[s][i][lane];
                finish(i, y);
            }
            __syncthreads();
            if (me.live)
                for (int i = slice; i < steps; i += k.slices) ((T*)a.out.p)[(t0 + i) * a.out.st + n * a.out.sn + me.c] = lx[i * kWave + lane];
        } else {
#pragma unroll
            for (int i = 0; i < SCAN_STEPS; i++) finish(i, u[i]);
            wave_wrote();
            const Scan& k = args_again();
            ChunkIn<T>::leave(lx, k.a.out, t0, steps, place.again(), k.wide);
        }
    }
    const ScanPlace& me = place;
    if (!me.live) return;
    if (SUMS) {
#pragma unroll
        for (int s = 0; s < SP; s++) k.seg_h[seg0 + (int64_t)s * a.C] = h[s];
        if (slice == 0) k.seg_d[(me.segment * a.N + n) * a.C + c] = total;
    } else if (last == k.chunks) {
        store_states<SP>(a, a.state_out, n, c, me.s0, h);
    }
}

// From what each segment adds to what enters each (in place; bound by the waits between segments: 126 of 2 envs, 1,024 channels of 16 states
// 18 us, 37 with one segment in flight): forwards in time from the state, or (BACK) backwards from its gradient.
template <bool BACK> __global__ void __launch_bounds__(256) k_scan_enter(Scan k) {
    const MoScan& a = k.a;
    const int64_t id = block_here() * 256 + threadIdx.x, row = id / a.C;
    if (row >= a.N * k.SB) return;
    const int c = (int)(id % a.C), s = (int)(row % k.SB);
    const int64_t n = row / k.SB;
    const bool real = s < a.S;
    const float* from = BACK ? a.dstate_out : a.state;
    const float A = real ? a.A[(int64_t)c * a.S + s] * LOG2E : 0.f;
    float h = from && real ? from[(n * a.C + c) * a.S + s] : 0.f;
    constexpr int IN_FLIGHT = 8;                              // segments whose values are read before they are joined
    const int64_t far = BACK ? k.segments - 1 : 0, to_d = (BACK ? -1 : 1) * a.N * a.C, to_h = to_d * k.SB;
    float* at = k.seg_h + ((far * a.N + n) * k.SB + s) * a.C + c;
    const float* size = k.seg_d + (far * a.N + n) * a.C + c;
    for (int64_t left = k.segments; left > 0; left -= IN_FLIGHT) {
        float add[IN_FLIGHT], d[IN_FLIGHT];
#pragma unroll
        for (int i = 0; i < IN_FLIGHT; i++) {
            const int64_t j = min((int64_t)i, left - 1);
            add[i] = at[j * to_h];
            d[i] = size[j * to_d];
        }
#pragma unroll
        for (int i = 0; i < IN_FLIGHT; i++) {
            if (i >= left) break;
            at[i * to_h] = h;
            h = d[i] < 0.f ? add[i] : fmaf(exp2_raw(d[i] * A), h, add[i]);
        }
        at += IN_FLIGHT * to_h;
        size += IN_FLIGHT * to_d;
    }
}

// ---- host side
struct ScanCut { int SP, slices; };
inline ScanCut scan_slices(int S) {
    const int slices = (S + 15) / 16, SP = ((S + slices - 1) / slices + 3) / 4 * 4;
    return {SP, slices};
}
constexpr int64_t SCAN_FILL = 4096;     // waves that fill the card
constexpr int SCAN_BACK_WAVES = 8;      // waves a workgroup of the gradient, at most
// LDS of a wave there: four tiles of values, three of float32, sums for dB and dC, dA; more where it shares its channels.
constexpr int scan_back_lds(int size, int SP, bool split) {
    constexpr int TILE = SCAN_STEPS * kWave;
    return 4 * TILE * size + 4 * (3 * TILE + (split ? 1 : 2) * SCAN_STEPS * 32 + SP * kWave + (size == 4 ? 0 : TILE) + (!split ? 0 : size == 4 ? TILE : 2 * TILE));
}
inline Scan scan_cut(const MoScan& a, bool backward) {
    Scan k{};
    k.a = a;
    const ScanCut c = scan_slices(a.S);
    k.slices = c.slices;
    k.SB = c.SP * c.slices;
    k.Cg = a.C / a.G;
    k.per = (k.Cg + kWave - 1) / kWave;
    // Rows in pieces, where their places in a chunk fit 32 bits: steps of up to 2^27 elements in bf16, 2^26 in float32 (16 steps of 32,768 envs, 512 channels of
    // 16 states, gated by half of a projection of 1,024: 1,571 us; rows an element a lane, 1,721).
    const int64_t V = a.dtype == MO_BF16 ? 8 : 4, farthest = ((int64_t)1 << 31) / (SCAN_STEPS * (16 / V));
    const auto row = [&](const MoRows& r) { return !r.p || ((uintptr_t)r.p % 16 == 0 && r.st % V == 0 && r.sn % V == 0 && r.st >= 0 && r.st <= farthest); };
    k.wide = k.Cg % V == 0 && row(a.x) && row(a.dt) && row(a.z) && (backward ? row(a.dout) && row(a.dx) && row(a.ddt) && row(a.dz) : row(a.out));
    k.chunks = (a.T + SCAN_STEPS - 1) / SCAN_STEPS;
    const int lds = scan_back_lds(a.dtype == MO_BF16 ? 2 : 4, c.SP, k.slices > 1), room = (160 << 10) / lds;
    k.across = std::min(k.per, std::min(SCAN_BACK_WAVES, room) / k.slices);
    k.cuts = (k.per + k.across - 1) / k.across;
    // Few sequences are cut over their length: each segment is gone through twice, once for what it adds to the state. The forward pass has many waves a
    // compute unit and takes whatever number; the gradient has few, so its segments are as many as run at once (1,999 steps of 8 envs, 512
    // channels: 32 segments, 160 us; 50, which run in two rounds, 201). The forward pass is cut where four times its waves or more fill the card (512
    // channels of 16 states in bf16, cut and in one piece: 512 steps x 80 envs, six times, 194 us and 250; 128 envs, four times, 512 steps 271 and 253,
    // 1,999 steps 946 and 958; 170 envs, three times, 351 and 335), and a segment has four chunks at least (with two, four or eight: forward 128 x 8
    // 31, 43 and 68 us, 128 x 64 67, 62 and 74; forward and gradient by the gradient's segments, 300 x 8 145, 176 and 272, 1,999 x 8 329, 330 and 340).
    const int64_t waves = std::max<int64_t>(1, a.N * a.G * k.per * k.slices), most = std::max<int64_t>(1, SCAN_FILL / waves);
    const int block = k.across * k.slices;
    const int64_t at_once = std::max<int64_t>(1, 256 * std::max(1, std::min((160 << 10) / (block * lds), (c.SP > 8 ? 8 : 12) / block)) / (a.G * k.cuts));
    const int64_t want = backward ? at_once / std::max<int64_t>(1, a.N) : most >= 4 ? most : 1;
    k.segments = std::max<int64_t>(1, std::min(want, k.chunks / 4));
    k.each = std::max<int64_t>(1, (k.chunks + k.segments - 1) / k.segments);
    k.segments = std::max<int64_t>(1, (k.chunks + k.each - 1) / k.each);
    if (backward) {   // as many at a time as run at once, and about the same number of turns for each
        const int64_t items = k.segments * a.N, turns = std::max<int64_t>(1, (items + at_once - 1) / at_once);
        k.rows = (items + turns - 1) / turns;
    }
    return k;
}
// In floats, each part a multiple of 4 of them.
inline int64_t whole(int64_t n) { return (n + 3) / 4 * 4; }
inline int64_t scan_bc(const Scan& k) { return whole(scan_rows(k) * k.a.N * k.a.G * 2 * k.SB); }
inline int64_t scan_kept(const Scan& k) { return whole(k.chunks * k.a.N * k.SB * k.a.C); }
inline int64_t scan_segs(const Scan& k) { return k.segments > 1 ? whole(k.segments * k.a.N * (k.SB + 1) * k.a.C) : 0; }
inline int64_t scan_parts_bc(const Scan& k) { return k.cuts > 1 ? whole(k.cuts * k.a.T * k.a.N * k.a.G * 2 * k.SB) : 0; }
inline int64_t scan_parts(const Scan& k) { return whole(k.rows * (k.SB + 2) * k.a.C); }
inline int64_t scan_work_floats(const Scan& k, bool backward) {
    if (!backward) return (k.a.saved ? 0 : scan_bc(k)) + scan_segs(k);
    return scan_segs(k) + scan_parts_bc(k) + scan_parts(k) + column_sums_work(k.rows, k.SB + 2, k.a.C);
}

// f(states a lane, whether waves share channels, whether some of the states are not there)
template <class F> int by_states(const Scan& k, F f) {
    const int SP = k.SB / k.slices;
    const auto padded = [&](auto sp, auto split) { return k.SB == k.a.S ? f(sp, split, std::false_type{}) : f(sp, split, std::true_type{}); };
    if (k.slices == 1) {
        if (SP == 4) return padded(std::integral_constant<int, 4>{}, std::false_type{});
        if (SP == 8) return padded(std::integral_constant<int, 8>{}, std::false_type{});
        if (SP == 12) return padded(std::integral_constant<int, 12>{}, std::false_type{});
        return padded(std::integral_constant<int, 16>{}, std::false_type{});
    }
    if (SP == 12) return padded(std::integral_constant<int, 12>{}, std::true_type{});
    return padded(std::integral_constant<int, 16>{}, std::true_type{});
}
inline void scan_launch_shape(const Scan& k, int64_t waves, dim3& grid, dim3& block) {
    grid = grid_of(k.slices > 1 ? waves : (waves + SCAN_WAVES - 1) / SCAN_WAVES);
    block = dim3(kWave * (k.slices > 1 ? k.slices : SCAN_WAVES));
}

template <class T> int scan_forward(const MoScan& a, hipStream_t s) {
    Scan k = scan_cut(a, false);
    float* bc = (float*)(a.saved ? a.saved : a.work);
    k.bc = bc;
    k.kept = a.saved ? bc + scan_bc(k) : nullptr;
    k.seg_h = (float*)a.work + (a.saved ? 0 : scan_bc(k));
    k.seg_d = k.seg_h + k.segments * a.N * k.SB * a.C;
    if (a.T) {
        const int64_t n = scan_rows(k) * a.N * a.G * (k.SB / 2);
        hipLaunchKernelGGL((k_scan_pack<T>), grid_of((n + 255) / 256), dim3(256), 0, s, k, bc);
        if (launched("k_scan_pack")) return -1;
    }
    return by_states(k, [&](auto sp, auto split, auto pad) {
        constexpr int SP = decltype(sp)::value;
        constexpr bool SPLIT = decltype(split)::value, PAD = decltype(pad)::value;
        dim3 grid, block;
        scan_launch_shape(k, k.segments * a.N * a.G * k.per, grid, block);
        if (k.segments > 1) {
            hipLaunchKernelGGL((k_scan<T, SP, SPLIT, true, false>), grid, block, 0, s, k);
            hipLaunchKernelGGL((k_scan_enter<false>), grid_of((a.N * k.SB * a.C + 255) / 256), dim3(256), 0, s, k);
        }
        hipLaunchKernelGGL((k_scan<T, SP, SPLIT, false, PAD>), grid, block, 0, s, k);
        return launched("k_scan");
    });
}

}  // namespace mo
