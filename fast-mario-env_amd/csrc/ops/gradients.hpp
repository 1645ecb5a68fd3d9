// The norm of many tensors together, and their scaling by it.
#pragma once
#include "common.hpp"

namespace mo {

// The tensors go into the kernels' arguments, up to GRADIENT_TABLE of them a launch. A workgroup takes every gridDim.x-th chunk of the launch's
// values and leaves one float64 sum of squares; the scaling kernel's workgroups each add all of these, in the same order, and go through the
// chunks backwards: what was read last is still in the last-level cache. Bound by memory: 201 tensors of 150M float32 148 + 206 us (4.0 TB/s read, 5.8 read
// and written; 328 + 429 in 4-byte accesses); 22 tensors of 2.7M values 5 + 10, of them the host's checks and launches take 19. A chunk is read in 16-byte accesses from the first value that lies on 16 bytes.
constexpr int GRADIENT_TABLE = 240, GRADIENT_THREADS = 256, GRADIENT_BLOCKS = 2048;
constexpr int64_t GRADIENT_CHUNK = 4096;    // values of the smallest chunk
struct Gradients {
    void* p[GRADIENT_TABLE];
    uint32_t begin[GRADIENT_TABLE + 1];   // the first chunk of each tensor
    uint32_t last[GRADIENT_TABLE];        // values of its last chunk; the top bit: bf16
    int count, chunk;
};
static_assert(sizeof(Gradients) < 3900, "");   // (a launch's arguments are 4 KB)

__device__ __forceinline__ int tensor_of(const Gradients& g, unsigned chunk) {
    int lo = 0, hi = g.count - 1;          // the last tensor that begins at or before the chunk
    while (lo < hi) {
        const int mid = (lo + hi + 1) / 2;
        if (g.begin[mid] <= chunk) lo = mid;
        else hi = mid - 1;
    }
    return lo;
}
__device__ __forceinline__ double block_sum(double x, double* s) {
    for (int m = kWave / 2; m; m /= 2) x += __shfl_xor(x, m);
    __syncthreads();
    if (threadIdx.x % kWave == 0) s[threadIdx.x / kWave] = x;
    __syncthreads();
    x = 0.0;
    for (int w = 0; w < GRADIENT_THREADS / kWave; w++) x += s[w];
    return x;
}

struct GradientChunk {
    void* p;
    int n;
    bool bf;
    __device__ __forceinline__ GradientChunk(const Gradients& g, unsigned chunk) {
        const int i = tensor_of(g, chunk);
        const int64_t at = (int64_t)(chunk - g.begin[i]) * g.chunk;
        bf = g.last[i] >> 31;
        n = chunk + 1 < g.begin[i + 1] ? g.chunk : (int)(g.last[i] & 0x7fffffffu);
        p = bf ? (void*)((bf16*)g.p[i] + at) : (void*)((float*)g.p[i] + at);
    }
};
// f(a value's place, 16 bytes or one value) over the chunk's values; IN_FLIGHT accesses a thread before the first is used.
constexpr int GRADIENT_IN_FLIGHT = 4;
template <class T, class Wide, class One> __device__ __forceinline__ void over_chunk(T* p, int n, Wide wide, One one) {
    constexpr int V = 16 / sizeof(T);
    const int head = min(n, (int)((-(uintptr_t)p & 15) / sizeof(T))), packs = (n - head) / V, tail = head + packs * V;
    if ((int)threadIdx.x < head) one(p + threadIdx.x);
    typedef Pack<std::remove_const_t<T>, V> P;
    P* at = (P*)(uintptr_t)(p + head);
    int i = threadIdx.x;
    for (; i + (GRADIENT_IN_FLIGHT - 1) * GRADIENT_THREADS < packs; i += GRADIENT_IN_FLIGHT * GRADIENT_THREADS) {
        P x[GRADIENT_IN_FLIGHT];
#pragma unroll
        for (int j = 0; j < GRADIENT_IN_FLIGHT; j++) x[j] = at[i + j * GRADIENT_THREADS];
#pragma unroll
        for (int j = 0; j < GRADIENT_IN_FLIGHT; j++) wide(at + i + j * GRADIENT_THREADS, x[j]);
    }
    for (; i < packs; i += GRADIENT_THREADS) wide(at + i, at[i]);
    if (tail + (int)threadIdx.x < n) one(p + tail + threadIdx.x);
}
template <class T> __device__ __forceinline__ double squares(const T* p, int n) {
    double x = 0.0;
    const auto add = [&](T y) {
        const double v = as_f32(y);
        x = fma(v, v, x);
    };
    over_chunk(p, n, [&](const auto*, const auto& y) {
#pragma unroll
        for (int v = 0; v < (int)(16 / sizeof(T)); v++) add(y.v[v]);
    }, [&](const T* y) { add(*y); });
    return x;
}
__global__ void __launch_bounds__(GRADIENT_THREADS) k_gradient_squares(Gradients g, double* part) {
    __shared__ double s[GRADIENT_THREADS / kWave];
    double x = 0.0;
    for (unsigned chunk = blockIdx.x; chunk < g.begin[g.count]; chunk += gridDim.x) {
        const GradientChunk c(g, chunk);
        x += c.bf ? squares((const bf16*)c.p, c.n) : squares((const float*)c.p, c.n);
    }
    x = block_sum(x, s);
    if (threadIdx.x == 0) part[blockIdx.x] = x;
}

__device__ __forceinline__ double norm_of(const double* part, int64_t parts, double* s) {
    double x = 0.0;
    for (int64_t i = threadIdx.x; i < parts; i += GRADIENT_THREADS) x += part[i];
    return sqrt(block_sum(x, s));
}
__global__ void __launch_bounds__(GRADIENT_THREADS) k_gradient_norm(const double* part, int64_t parts, float* norm) {
    __shared__ double s[GRADIENT_THREADS / kWave];
    const double x = norm_of(part, parts, s);
    if (threadIdx.x == 0) *norm = (float)x;
}
template <class T> __device__ __forceinline__ void scale_values(T* p, int n, float by) {
    over_chunk(p, n, [&](auto* to, auto y) {
#pragma unroll
        for (int v = 0; v < (int)(16 / sizeof(T)); v++) y.v[v] = as<T>(as_f32(y.v[v]) * by);
        stream(to, y);
    }, [&](T* y) { *y = as<T>(as_f32(*y) * by); });
}
// (max / (norm + eps) is taken in float64 and the factor rounded once to float32; a norm that is NaN makes everything NaN.)
__global__ void __launch_bounds__(GRADIENT_THREADS) k_gradient_scale(Gradients g, const double* part, int64_t parts, float max_norm, float eps, float* norm) {
    __shared__ double s[GRADIENT_THREADS / kWave];
    const double x = norm_of(part, parts, s), f = (double)max_norm / (x + (double)eps);
    if (norm && blockIdx.x == 0 && threadIdx.x == 0) *norm = (float)x;
    const float by = f > 1.0 ? 1.f : (float)f;
    const unsigned chunks = g.begin[g.count];
    for (unsigned back = blockIdx.x; back < chunks; back += gridDim.x) {
        const GradientChunk c(g, chunks - 1 - back);
        if (c.bf) scale_values((bf16*)c.p, c.n, by);
        else scale_values((float*)c.p, c.n, by);
    }
}

// ---- host side
inline int64_t gradient_launches(int64_t count) { return std::max<int64_t>(1, (count + GRADIENT_TABLE - 1) / GRADIENT_TABLE); }
inline int64_t gradient_work(int64_t count) { return 8 * gradient_launches(count) * GRADIENT_BLOCKS; }
inline int gradient_norm(const MoTensor* t, int64_t count, bool scale, float max_norm, float eps, float* norm, double* part, hipStream_t s) {
    const int64_t launches = gradient_launches(count);
    int64_t values = 0;
    for (int64_t i = 0; i < count; i++) values += t[i].n;
    const int64_t chunk = GRADIENT_CHUNK * std::clamp<int64_t>(values / (GRADIENT_CHUNK * GRADIENT_BLOCKS), 1, 16);
    const auto table = [&](int64_t l, Gradients& g) {
        g = Gradients{};
        g.chunk = (int)chunk;
        uint64_t chunks = 0;
        for (int64_t i = l * GRADIENT_TABLE; i < std::min(count, (l + 1) * GRADIENT_TABLE); i++) {
            if (!t[i].n) continue;
            const int k = g.count++;
            const int64_t of = (t[i].n + chunk - 1) / chunk;
            g.p[k] = t[i].p;
            g.begin[k] = (uint32_t)chunks;
            g.last[k] = (uint32_t)(t[i].n - (of - 1) * chunk) | (t[i].dtype == MO_BF16 ? 1u << 31 : 0u);
            chunks += of;
        }
        g.begin[g.count] = (uint32_t)chunks;
        return (unsigned)std::min<uint64_t>(std::max<uint64_t>(chunks, 1), GRADIENT_BLOCKS);
    };
    Gradients g;
    int64_t parts = 0;
    for (int64_t l = 0; l < launches; l++) {
        const unsigned blocks = table(l, g);
        hipLaunchKernelGGL(k_gradient_squares, dim3(blocks), dim3(GRADIENT_THREADS), 0, s, g, part + parts);
        parts += blocks;
    }
    if (launched("k_gradient_squares")) return -1;
    if (!scale) {
        hipLaunchKernelGGL(k_gradient_norm, dim3(1), dim3(GRADIENT_THREADS), 0, s, (const double*)part, parts, norm);
        return launched("k_gradient_norm");
    }
    for (int64_t l = launches - 1; l >= 0; l--) {
        const unsigned blocks = table(l, g);
        hipLaunchKernelGGL(k_gradient_scale, dim3(blocks), dim3(GRADIENT_THREADS), 0, s, g, (const double*)part, parts, max_norm, eps, l ? nullptr : norm);
    }
    return launched("k_gradient_scale");
}

}  // namespace mo
