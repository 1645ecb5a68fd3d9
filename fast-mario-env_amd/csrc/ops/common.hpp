// What the policy's operators share: element types, wave reductions, and the host's checks and errors.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <algorithm>
#include <stdexcept>
#include <string>

#include "../../../include/mario_ops.h"

namespace mo {

typedef __bf16 bf16;

__device__ __forceinline__ float as_f32(float x) { return x; }
__device__ __forceinline__ float as_f32(bf16 x) { return (float)x; }
// The one rounding of a value to the type it is stored in (to nearest even).
template <class T> __device__ __forceinline__ T as(float x) { return (T)x; }

// N consecutive elements as they lie in memory, moved in accesses of up to 16 bytes.
template <class T, int N> struct alignas(sizeof(T) * N > 16 ? 16 : sizeof(T) * N) Pack { T v[N]; };

constexpr int kWave = 64;

// A launch has fewer than 2^32 threads along x: past 2^22 blocks it goes on along z. Blocks past the last one have nothing to do.
constexpr int kGridBits = 22;
__device__ __forceinline__ int64_t block_here() { return ((int64_t)blockIdx.z << kGridBits) + blockIdx.x; }
inline dim3 grid_of(int64_t blocks, int64_t y = 1) {
    const int64_t x = std::min(blocks, (int64_t)1 << kGridBits);
    return dim3((unsigned)x, (unsigned)y, (unsigned)((blocks + x - 1) / x));
}

// What is larger than the last-level cache and read once comes past the caches' reuse order.
constexpr int64_t LAST_LEVEL_CACHE = 256 << 20;
template <class P> __device__ __forceinline__ P streamed(const P* from) {
    P x;
    if constexpr (sizeof(P) == 16) {
        typedef unsigned U __attribute__((ext_vector_type(4)));
        *(U*)&x = __builtin_nontemporal_load((const U*)from);
    } else if constexpr (sizeof(P) == 32) {
        typedef unsigned U __attribute__((ext_vector_type(4)));
        ((U*)&x)[0] = __builtin_nontemporal_load((const U*)from);
        ((U*)&x)[1] = __builtin_nontemporal_load((const U*)from + 1);
    } else if constexpr (sizeof(P) == 4) {
        *(unsigned*)&x = __builtin_nontemporal_load((const unsigned*)from);
    } else {
        x = *from;
    }
    return x;
}

// What is written once, in whole cache lines, leaves past the caches' reuse order (nontemporal). In bf16, with plain stores instead: group
// norm of 500 x 32 x 84 x 84 118 and 149 us, forward and gradient of 16,384 x 32 x 9 x 9 in 4 groups 95 and 106; a single step of 32,768 envs
// 1,439 and 1,527; linear attention 1 to 3 % (128 steps of 4,096 envs 754 and 766), where heads of 40, which fill no lines, lose 4 %.
template <class P> __device__ __forceinline__ void stream(P* to, const P& x) {
    if constexpr (sizeof(P) == 16) {
        typedef unsigned U __attribute__((ext_vector_type(4), aligned(4)));   // (aligned to elements is enough)
        __builtin_nontemporal_store(*(const U*)&x, (U*)to);
    } else if constexpr (sizeof(P) == 32) {
        typedef unsigned U __attribute__((ext_vector_type(4)));
        __builtin_nontemporal_store(((const U*)&x)[0], (U*)to);
        __builtin_nontemporal_store(((const U*)&x)[1], (U*)to + 1);
    } else if constexpr (sizeof(P) == 8) {
        typedef unsigned U __attribute__((ext_vector_type(2)));
        __builtin_nontemporal_store(*(const U*)&x, (U*)to);
    } else if constexpr (sizeof(P) == 4) {
        __builtin_nontemporal_store(*(const unsigned*)&x, (unsigned*)to);
    } else {
        *to = x;
    }
}

// ---- host side
inline thread_local std::string g_err;

inline int fail(const std::string& what) {
    g_err = what;
    return -1;
}
inline bool ok(hipError_t e, const char* what) {
    if (e == hipSuccess) return true;
    fail(std::string(what) + ": " + hipGetErrorString(e));
    return false;
}
inline int launched(const char* what) { return ok(hipGetLastError(), what) ? 0 : -1; }

// A buffer a kernel is about to touch: memory of the current GPU (device, pinned host or managed), aligned to its
// elements. Anything else is refused before a kernel could fault on it.
inline bool usable(const void* p, const char* name, size_t align) {
    if (!p) { fail(std::string(name) + ": null"); return false; }
    if ((uintptr_t)p % align) { fail(std::string(name) + ": not aligned to its elements"); return false; }
    int dev = 0;
    if (!ok(hipGetDevice(&dev), "hipGetDevice")) return false;
    hipPointerAttribute_t at;
    const hipError_t e = hipPointerGetAttributes(&at, p);
    (void)hipGetLastError();   // a refused pointer must not surface as the error of a later launch
    const bool good = e == hipSuccess && ((at.type == hipMemoryTypeDevice && at.device == dev) ||
                                          at.type == hipMemoryTypeHost || at.type == hipMemoryTypeManaged);
    if (!good) fail(std::string(name) + ": not memory of GPU " + std::to_string(dev));
    return good;
}

inline int compute_units() {
    int dev = 0, cus = 0;
    if (hipGetDevice(&dev) != hipSuccess ||
        hipDeviceGetAttribute(&cus, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess || cus < 1) return 256;
    return cus;
}

}  // namespace mo
