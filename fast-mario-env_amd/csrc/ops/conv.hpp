// Causal convolution over the steps of each channel, with an activation: forward, gradient and single step.
#pragma once
#include "sums.hpp"

namespace mo {

constexpr int CONV_THREADS = 256;
// (Gradient) steps whose loads are in flight: as many as leave two waves a SIMD (128 x 2,048 x 512 bf16, K = 4: 258 us with one, 225 with two).
template <int V> constexpr int CONV_AHEAD = V > 4 ? 2 : 4;

// A thread holds V neighbouring channels of one env and goes through a segment of the steps with the last K - 1 inputs in registers, cleared where an
// episode starts; segments begin by reading the K - 1 steps before them. The forward pass is bound by memory (128 x 2,048 x 512 bf16: 107 us, 5.0
// TB/s), the gradient by the vector units (195 to 215 us, 91 % busy: 40 instructions a value, the argument made again among them).
struct Conv {
    MoConv a;
    int64_t each, segments;    // steps of a segment
    int64_t rows;              // (gradient) segments of envs that are taken at a time
    float* part;               // (gradient) (rows, K + 1, C): each row's sums for dweight and dbias
};

template <int ACT> __device__ __forceinline__ float act_of(float p) {
    if (ACT == MO_ACT_RELU) return p <= 0.f ? 0.f : p;   // (a NaN stays one, and its gradient goes on)
    if (ACT == MO_ACT_SILU) return p * __builtin_amdgcn_rcpf(1.f + __expf(-p));
    return p;
}
template <int ACT> __device__ __forceinline__ float act_slope(float p) {
    if (ACT == MO_ACT_RELU) return p <= 0.f ? 0.f : 1.f;
    if (ACT == MO_ACT_SILU) {
        const float s = __builtin_amdgcn_rcpf(1.f + __expf(-p));
        return s * fmaf(p, 1.f - s, 1.f);
    }
    return 1.f;
}

template <class T, int V> __device__ __forceinline__ void load_channels(float (&x)[V], const T* p) {
    const Pack<T, V> y = *(const Pack<T, V>*)p;
#pragma unroll
    for (int c = 0; c < V; c++) x[c] = as_f32(y.v[c]);
}
template <class T, int V> __device__ __forceinline__ void store_channels(T* p, const float (&x)[V]) {
    Pack<T, V> y;
#pragma unroll
    for (int c = 0; c < V; c++) y.v[c] = as<T>(x[c]);
    *(Pack<T, V>*)p = y;
}
template <class T> __device__ __forceinline__ T* row_at(const MoRows& r, int64_t t, int64_t n) { return (T*)r.p + t * r.st + n * r.sn; }

template <int V, int K> __device__ __forceinline__ void load_taps(const MoConv& a, int c, float (&w)[K][V], float (&b)[V]) {
#pragma unroll
    for (int v = 0; v < V; v++) {
#pragma unroll
        for (int k = 0; k < K; k++) w[k][v] = a.weight[(int64_t)(c + v) * K + k];
        b[v] = a.bias ? a.bias[c + v] : 0.f;
    }
}
// The K - 1 inputs before step t0, newest first, 0 where step t0 - 1's episode does not hold them.
template <class T, int V, int K> __device__ __forceinline__ void load_window(const MoConv& a, int64_t t0, int64_t n, int c, float (&win)[K][V]) {
    bool alive = true;
#pragma unroll
    for (int j = 1; j < K; j++) {
        const int64_t t = t0 - j;
#pragma unroll
        for (int v = 0; v < V; v++) win[j - 1][v] = 0.f;
        if (!alive) continue;
        if (t >= 0) {
            load_channels<T, V>(win[j - 1], row_at<T>(a.x, t, n) + c);
            alive = !(a.start && a.start[t * a.N + n]);
        } else if (a.state) {
            load_channels<T, V>(win[j - 1], (const T*)a.state + (n * (K - 1) + (K - 1 + t)) * a.C + c);
        }
    }
}

template <class T, int V, int K, int ACT>
__global__ void __launch_bounds__(CONV_THREADS) k_conv(Conv k) {
    const MoConv& a = k.a;
    const int lanes = a.C / V;
    const int64_t id = block_here() * CONV_THREADS + threadIdx.x, row = id / lanes;
    const int c = (int)(id % lanes) * V;
    if (row >= k.segments * a.N) return;
    const int64_t n = row % a.N, t0 = row / a.N * k.each, t1 = min(a.T, t0 + k.each);
    float w[K][V], b[V], win[K][V];
    load_taps<V, K>(a, c, w, b);
    load_window<T, V, K>(a, t0, n, c, win);
    const T* from = row_at<T>(a.x, t0, n) + c;               // (moved on from step to step: no products of 64 bits between them)
    T* to = row_at<T>(a.y, t0, n) + c;
    const uint8_t* flag = a.start ? a.start + t0 * a.N + n : nullptr;
    for (int64_t t = t0; t < t1; t++, from += a.x.st, to += a.y.st) {
        float x[V], p[V];
        load_channels<T, V>(x, from);
        const bool cut = flag && *flag;
        if (flag) flag += a.N;
#pragma unroll
        for (int v = 0; v < V; v++) {
            p[v] = fmaf(w[K - 1][v], x[v], b[v]);
#pragma unroll
            for (int j = 1; j < K; j++) {
                win[j - 1][v] = cut ? 0.f : win[j - 1][v];
                p[v] = fmaf(w[K - 1 - j][v], win[j - 1][v], p[v]);
            }
            p[v] = act_of<ACT>(p[v]);
#pragma unroll
            for (int j = K - 1; j > 1; j--) win[j - 1][v] = win[j - 2][v];
            if (K > 1) win[0][v] = x[v];
        }
        store_channels<T, V>(to, p);
    }
    if (t1 != a.T || !a.state_out) return;
#pragma unroll
    for (int j = 1; j < K; j++) store_channels<T, V>((T*)a.state_out + (n * (K - 1) + (K - 1 - j)) * a.C + c, win[j - 1]);
}

// The gradient of step t's argument, dp_t, goes to the K inputs that it saw. Those of steps not yet complete wait in registers: that of step t - j in
// wait[j]. Where an episode starts, what waits is complete and leaves at once; `age` counts the steps since, so that nothing leaves
// twice. A segment goes K - 1 steps past its end, for its own last inputs. Inputs before step 0 are the entering state's rows.
template <class T, int V, int K, int ACT>
__global__ void __launch_bounds__(CONV_THREADS, 2) k_conv_back(Conv k) {
    const MoConv& a = k.a;
    constexpr int AHEAD = CONV_AHEAD<V>;
    const int lanes = a.C / V;
    const int64_t id = block_here() * CONV_THREADS + threadIdx.x, first = id / lanes;
    const int c = (int)(id % lanes) * V;
    if (first >= k.rows) return;
    float w[K][V], b[V], dw[K][V], db[V];
    load_taps<V, K>(a, c, w, b);
#pragma unroll
    for (int v = 0; v < V; v++) {
        db[v] = 0.f;
#pragma unroll
        for (int j = 0; j < K; j++) dw[j][v] = 0.f;
    }
    for (int64_t row = first; row < k.segments * a.N; row += k.rows) {
        const int64_t n = row % a.N, t0 = row / a.N * k.each, t1 = min(a.T, t0 + k.each), past = min(a.T, t1 + K - 1);
        const int64_t own = t0 ? t0 : 1 - K;                  // the first input whose gradient is this segment's
        float win[K][V], wait[K][V];
        load_window<T, V, K>(a, t0, n, c, win);
#pragma unroll
        for (int j = 0; j < K; j++)
#pragma unroll
            for (int v = 0; v < V; v++) wait[j][v] = 0.f;
        const auto leave = [&](int64_t t, const float (&x)[V]) {
            if (t < own || t >= t1) return;
            if (t >= 0) store_channels<T, V>(row_at<T>(a.dx, t, n) + c, x);
            else if (a.dstate) store_channels<T, V>((T*)a.dstate + (n * (K - 1) + (K - 1 + t)) * a.C + c, x);
        };
        int age = K - 2;
        Pack<T, V> px[AHEAD], pdy[AHEAD];
        uint8_t pcut[AHEAD];
        const T *from_x = row_at<T>(a.x, t0, n) + c, *from_dy = row_at<T>(a.dy, t0, n) + c;
        T* to = row_at<T>(a.dx, t0 - (K - 1), n) + c;
        const uint8_t* flag = a.start ? a.start + t0 * a.N + n : nullptr;
        const auto ahead = [&](int i) {
            px[i] = *(const Pack<T, V>*)from_x;
            pdy[i] = *(const Pack<T, V>*)from_dy;
            pcut[i] = flag ? *flag : 0;
            from_x += a.x.st;
            from_dy += a.dy.st;
            if (flag) flag += a.N;
        };
#pragma unroll
        for (int i = 0; i < AHEAD; i++)
            if (t0 + i < past) ahead(i);
        const auto step = [&](int64_t t, int i) {
            float x[V], dy[V];
#pragma unroll
            for (int v = 0; v < V; v++) {
                x[v] = as_f32(px[i].v[v]);
                dy[v] = as_f32(pdy[i].v[v]);
            }
            const bool cut = pcut[i];
            if (t + AHEAD < past) ahead(i);
            if (cut) {
#pragma unroll
                for (int j = 1; j < K; j++) {
                    if (j <= age + 1) leave(t - j, wait[j]);
#pragma unroll
                    for (int v = 0; v < V; v++) win[j - 1][v] = 0.f;
                }
                age = 0;
            } else {
                age = min(age + 1, K);
            }
            const bool mine = t < t1;
#pragma unroll
            for (int v = 0; v < V; v++) {
                float p = fmaf(w[K - 1][v], x[v], b[v]);
#pragma unroll
                for (int j = 1; j < K; j++) p = fmaf(w[K - 1 - j][v], win[j - 1][v], p);
                const float dp = dy[v] * act_slope<ACT>(p);
                wait[0][v] = 0.f;
#pragma unroll
                for (int j = 0; j < K; j++) wait[j][v] = fmaf(w[K - 1 - j][v], dp, wait[j][v]);
                if (mine) {
                    db[v] += dp;
                    dw[K - 1][v] = fmaf(dp, x[v], dw[K - 1][v]);
#pragma unroll
                    for (int j = 1; j < K; j++) dw[K - 1 - j][v] = fmaf(dp, win[j - 1][v], dw[K - 1 - j][v]);
                }
            }
            if (age >= K - 1) {
                const int64_t done = t - (K - 1);
                if (done >= 0 && done >= own) store_channels<T, V>(to, wait[K - 1]);   // (at most t1 - 1)
                else leave(done, wait[K - 1]);
            }
#pragma unroll
            for (int v = 0; v < V; v++) {
#pragma unroll
                for (int j = K - 1; j > 0; j--) wait[j][v] = wait[j - 1][v];
#pragma unroll
                for (int j = K - 1; j > 1; j--) win[j - 1][v] = win[j - 2][v];
                if (K > 1) win[0][v] = x[v];
            }
            to += a.dx.st;
        };
        for (int64_t t = t0; t < past; t += AHEAD)
#pragma unroll
            for (int i = 0; i < AHEAD; i++)
                if (t + i < past) step(t + i, i);
        if (past == a.T)                                      // the last steps' inputs are what is left, and the state after them
#pragma unroll
            for (int j = 1; j < K; j++) {
                if (j > age + 1) continue;
                if (a.dstate_out) {
                    float ds[V];
                    load_channels<T, V>(ds, (const T*)a.dstate_out + (n * (K - 1) + (K - 1 - j)) * a.C + c);
#pragma unroll
                    for (int v = 0; v < V; v++) wait[j][v] += ds[v];
                }
                leave(a.T - j, wait[j]);
            }
    }
    if (!k.part) return;
    float* to = k.part + first * (K + 1) * a.C + c;
#pragma unroll
    for (int j = 0; j < K; j++) store_channels<float, V>(to + (int64_t)j * a.C, dw[j]);
    store_channels<float, V>(to + (int64_t)K * a.C, db);
}

// One step: the window is the state, which moves on by one. A thread goes through E envs with the same taps, whose windows it has in flight
// together. Bound by memory: 32,768 envs, 512 channels, four taps, bf16 64 us, 4.2 TB/s (45 where the windows are still in the last-level cache); with
// an env a thread, whose taps are as much to read as its window, 82 (76).
template <class T, int V, int K, int ACT, int E>
__global__ void __launch_bounds__(CONV_THREADS) k_conv_step(MoConv a) {
    const int lanes = a.C / V;
    const int64_t id = block_here() * CONV_THREADS + threadIdx.x, n0 = id / lanes * E;
    const int c = (int)(id % lanes) * V;
    if (n0 >= a.N) return;
    typedef Pack<T, V> P;
    P win[E][K], x[E];
    bool cut[E];
#pragma unroll
    for (int e = 0; e < E; e++) {
        const int64_t n = min(n0 + e, a.N - 1);
        const T* state = (const T*)a.state_out + n * (K - 1) * a.C + c;
#pragma unroll
        for (int j = 1; j < K; j++) win[e][j - 1] = *(const P*)(state + (K - 1 - j) * (int64_t)a.C);
        x[e] = *(const P*)(row_at<T>(a.x, 0, n) + c);
        cut[e] = a.start && a.start[n];
    }
    float w[K][V], b[V];
    load_taps<V, K>(a, c, w, b);
#pragma unroll
    for (int e = 0; e < E; e++) {
        const int64_t n = n0 + e;
        if (n >= a.N) break;
        if (cut[e])
#pragma unroll
            for (int j = 1; j < K; j++) win[e][j - 1] = P{};
        float p[V];
#pragma unroll
        for (int v = 0; v < V; v++) {
            p[v] = fmaf(w[K - 1][v], as_f32(x[e].v[v]), b[v]);
#pragma unroll
            for (int j = 1; j < K; j++) p[v] = fmaf(w[K - 1 - j][v], as_f32(win[e][j - 1].v[v]), p[v]);
            p[v] = act_of<ACT>(p[v]);
        }
        store_channels<T, V>(row_at<T>(a.y, 0, n) + c, p);
        T* state = (T*)a.state_out + n * (K - 1) * a.C + c;
        if (K > 1) *(P*)(state + (K - 2) * (int64_t)a.C) = x[e];
#pragma unroll
        for (int j = 2; j < K; j++) *(P*)(state + (K - 1 - j) * (int64_t)a.C) = win[e][j - 2];
    }
}

// ---- host side
// Whole 16-byte pieces of channels, or one channel a thread.
inline bool conv_wide(const MoConv& a, bool backward, bool step) {
    const size_t z = a.dtype == MO_BF16 ? 2 : 4;
    const int64_t V = 16 / z;
    const auto row = [&](const MoRows& r) { return (uintptr_t)r.p % 16 == 0 && (step || r.st % V == 0) && r.sn % V == 0; };
    const auto at = [](const void* p) { return (uintptr_t)p % 16 == 0; };
    return a.C % V == 0 && row(a.x) && at(a.state) && (backward ? row(a.dy) && row(a.dx) && at(a.dstate_out) && at(a.dstate) : row(a.y) && at(a.state_out));
}
// Threads that fill the card; the gradient's have registers for two waves a SIMD (357 us for forward and gradient of 128 x 2,048 x 512, 368 with twice
// as many threads).
constexpr int64_t CONV_FILL = 256 * 1024, CONV_BACK_FILL = 256 * 512;
inline Conv conv_cut(const MoConv& a, int V, bool backward) {
    Conv k{};
    k.a = a;
    const int64_t lanes = std::max(1, a.C / V), fill = backward ? CONV_BACK_FILL : CONV_FILL, most = std::max<int64_t>(1, fill / std::max<int64_t>(1, lanes * a.N));
    // long segments where there are enough of them; the K - 1 steps before (and after) each are read again
    k.each = std::max<int64_t>(16, (a.T + most - 1) / most);
    k.segments = std::max<int64_t>(1, (a.T + k.each - 1) / k.each);
    k.rows = backward ? std::min(k.segments * a.N, std::max<int64_t>(1, fill / lanes)) : 0;
    return k;
}
// (The gradient's registers go by K and V: four channels a thread from five taps on.)
inline int conv_width(const MoConv& a, bool backward, bool step) {
    if (!conv_wide(a, backward, step)) return 1;
    return a.dtype == MO_BF16 && !(backward && a.K > 4) ? 8 : 4;
}
inline int64_t conv_back_work(const MoConv& a) {
    if (!a.dweight || a.N == 0) return 0;      // (without steps the sums are made all the same: zeros)
    const Conv k = conv_cut(a, conv_width(a, true, false), true);
    return 4 * (k.rows * (a.K + 1) * a.C + column_sums_work(k.rows, a.K + 1, a.C));
}

// RUN: 0 forward, 1 gradient, 2 step
template <class T, int V, int K, int ACT, int RUN> int conv_launch(const MoConv& a, hipStream_t s) {
    const int64_t lanes = a.C / V;
    const auto blocks = [&](int64_t rows) { return grid_of((rows * lanes + CONV_THREADS - 1) / CONV_THREADS); };
    if constexpr (RUN == 2) {
        constexpr int E = V > 1 ? 4 : 1;                      // (where there are threads enough all the same)
        if (E > 1 && a.N * lanes >= CONV_FILL) hipLaunchKernelGGL((k_conv_step<T, V, K, ACT, E>), blocks((a.N + E - 1) / E), dim3(CONV_THREADS), 0, s, a);
        else hipLaunchKernelGGL((k_conv_step<T, V, K, ACT, 1>), blocks(a.N), dim3(CONV_THREADS), 0, s, a);
        return launched("k_conv_step");
    } else {
        Conv k = conv_cut(a, V, RUN == 1);
        if constexpr (RUN == 0) {
            hipLaunchKernelGGL((k_conv<T, V, K, ACT>), blocks(k.segments * a.N), dim3(CONV_THREADS), 0, s, k);
            return launched("k_conv");
        } else {
            k.part = a.dweight ? (float*)a.work : nullptr;
            hipLaunchKernelGGL((k_conv_back<T, V, K, ACT>), blocks(k.rows), dim3(CONV_THREADS), 0, s, k);
            if (launched("k_conv_back") || !a.dweight) return launched("k_conv_back");
            ColumnSums c{(const float*)a.work, (float*)a.work + k.rows * (K + 1) * a.C, k.rows, K + 1, a.C, K, K, a.dweight, a.dbias, nullptr};
            return column_sums(c, s);
        }
    }
}
template <class T, int V, int RUN, int ACT, int K = 1, int LAST = MO_MAX_TAPS> int conv_taps(const MoConv& a, hipStream_t s) {
    if constexpr (K > LAST) return fail("taps");
    else return a.K == K ? conv_launch<T, V, K, ACT, RUN>(a, s) : conv_taps<T, V, RUN, ACT, K + 1, LAST>(a, s);
}

}  // namespace mo
