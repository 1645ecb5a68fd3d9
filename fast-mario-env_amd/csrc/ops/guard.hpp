// What the library's C entry points share.
#pragma once
#include "common.hpp"

namespace mo {

constexpr int64_t MAX_GRID = (int64_t)1 << 31;

inline size_t size_of(int dtype) { return dtype == MO_BF16 ? 2 : 4; }

template <class F> int by_type(int dtype, F f) { return dtype == MO_BF16 ? f(bf16{}) : f(float{}); }

template <class F> int by_act(int act, F f) {
    if (act == MO_ACT_RELU) return f(std::integral_constant<int, MO_ACT_RELU>{});
    if (act == MO_ACT_SILU) return f(std::integral_constant<int, MO_ACT_SILU>{});
    return f(std::integral_constant<int, MO_ACT_NONE>{});
}

// No C++ exception leaves a C entry point.
template <class F> auto guarded(F f) noexcept -> decltype(f()) {
    try {
        return f();
    } catch (...) {
        try { fail("out of host memory"); } catch (...) {}
        return -1;
    }
}

}  // namespace mo
