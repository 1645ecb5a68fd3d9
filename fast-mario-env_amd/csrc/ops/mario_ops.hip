// libmario_ops.so: the operators of a policy with a memory (include/mario_ops.h), gfx950. A library of its own: the emulator's
// is built for bit-exact float sums and scalar code, these for matrix instructions and memory.
#include <algorithm>

#include "attend_chunk_back.hpp"
#include "attend_step.hpp"
#include "attend_walk.hpp"
#include "common.hpp"
#include "norm_rows.hpp"
#include "norm_small.hpp"

using namespace mo;

namespace {

constexpr int64_t MAX_GRID = (int64_t)1 << 31;

size_t size_of(int dtype) { return dtype == MO_BF16 ? 2 : 4; }

bool attend_sizes(const MoAttend* a) {
    if (!a || (a->dtype != MO_F32 && a->dtype != MO_BF16) || a->T < 0 || a->N < 0 || a->H < 1 || a->D < 1 || a->D > MO_MAX_HEAD ||
        a->E < 1 || a->E > MO_MAX_HEAD) {
        fail("invalid arguments (dtype MO_F32 or MO_BF16, T >= 0, N >= 0, H >= 1, head sizes 1 .. 128)");
        return false;
    }
    if (a->N >= MAX_GRID / a->H || a->T > ((int64_t)1 << 40)) { fail("too many envs, heads or steps (N H < 2^31, T <= 2^40)"); return false; }
    return true;
}

bool rows_usable(const MoRows& r, const char* name, int dtype) { return usable(r.p, name, size_of(dtype)); }

bool norm_sizes(const MoNorm* a) {
    if (!a || (a->dtype != MO_F32 && a->dtype != MO_BF16) || a->act < MO_ACT_NONE || a->act > MO_ACT_SILU || a->B < 0 || a->S < 1 ||
        a->C < 1 || a->groups < 1 || a->C % a->groups || !(a->eps >= 0.f)) {
        fail("invalid arguments (dtype MO_F32 or MO_BF16, act MO_ACT_*, B >= 0, S >= 1, C a multiple of groups >= 1, eps >= 0)");
        return false;
    }
    if ((!a->weight) != (!a->bias)) { fail("weight and bias: both or neither"); return false; }
    if (a->C > (1 << 20) || a->S > ((int64_t)1 << 30) || a->B >= MAX_GRID / a->groups) {
        fail("too many samples, pixels or channels (C <= 2^20, S <= 2^30, B groups < 2^31)");
        return false;
    }
    return true;
}

template <class F> int by_type(int dtype, F f) { return dtype == MO_BF16 ? f(bf16{}) : f(float{}); }

// Heads in whole 16-byte pieces go by chunks on the matrix cores, the rest step by step.
template <class T> int attend_forward(const MoAttend& a, hipStream_t s) {
    if (!chunks_take(a, false)) return walk_forward<T>(a, s);
    const int p = padded_head(a);
    return p == 32 ? attend_chunks<T, 32>(a, s) : p == 64 ? attend_chunks<T, 64>(a, s) : attend_chunks<T, 128>(a, s);
}
template <class T> int attend_back(const MoAttend& a, hipStream_t s) {
    if (!chunks_take(a, true) || (!a.saved && attend_cut(a).chunks > 1)) return walk_backward<T>(a, s);
    const int p = padded_head(a);
    return p == 32 ? attend_back_chunks<T, 32>(a, s) : p == 64 ? attend_back_chunks<T, 64>(a, s) : attend_back_chunks<T, 128>(a, s);
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

template <class F> int by_act(int act, F f) {
    if (act == MO_ACT_RELU) return f(std::integral_constant<int, MO_ACT_RELU>{});
    if (act == MO_ACT_SILU) return f(std::integral_constant<int, MO_ACT_SILU>{});
    return f(std::integral_constant<int, MO_ACT_NONE>{});
}

int norm_run(const MoNorm& a, bool backward, hipStream_t s) {
    return by_type(a.dtype, [&](auto t) {
        typedef decltype(t) T;
        return by_act(a.act, [&](auto act) {
            constexpr int A = decltype(act)::value;
            SmallCut c;
            RowsCut r;
            if (norm_small_takes(a, backward, c)) return norm_small<T, A>(a, c, backward, s);
            if (norm_rows_takes(a, r)) return norm_rows<T, A>(a, r, backward, s);
            return norm_wide(a) ? norm_general<T, 8, A>(a, backward, s) : norm_general<T, 1, A>(a, backward, s);
        });
    });
}

int64_t norm_work(const MoNorm& a, bool backward) {
    SmallCut c;
    RowsCut r;
    if (norm_small_takes(a, backward, c)) return 4 * norm_small_work(a, c, backward);
    if (norm_rows_takes(a, r)) return 4 * norm_rows_work(a, r, backward);
    return 4 * norm_general_work(a, norm_cut(a, norm_wide(a) ? 8 : 1), backward).total;
}

}  // namespace

extern "C" {

const char* mo_last_error(void) { return g_err.c_str(); }

int64_t mo_attend_saved(const MoAttend* a) {
    return guarded([&]() -> int64_t {
        if (!attend_sizes(a)) return -1;
        return chunks_take(*a, false) ? saved_bytes(*a) : 0;
    });
}

int64_t mo_attend_work(const MoAttend* a, int backward) {
    return guarded([&]() -> int64_t {
        if (!attend_sizes(a)) return -1;
        return chunks_take(*a, backward) ? cut_bytes(*a, attend_cut(*a)) : 0;
    });
}

int mo_attend(const MoAttend* a, void* stream) {
    return guarded([&] {
        if (!attend_sizes(a)) return -1;
        if (a->N == 0) return 0;
        if (a->T && !(rows_usable(a->q, "q", a->dtype) && rows_usable(a->k, "k", a->dtype) && rows_usable(a->v, "v", a->dtype) &&
                      rows_usable(a->out, "out", a->dtype)))
            return -1;
        if (!usable(a->decay, "decay", 4) || !usable(a->state_out, "state_out", 4) || (a->state && !usable(a->state, "state", 4)) ||
            (a->T && a->start && !usable(a->start, "start", 1)))
            return -1;
        if (mo_attend_work(a, 0) > 0 && !usable(a->work, "work", 16)) return -1;
        if (a->saved && mo_attend_saved(a) > 0 && !usable(a->saved, "saved", 16)) return -1;
        return by_type(a->dtype, [&](auto t) { return attend_forward<decltype(t)>(*a, (hipStream_t)stream); });
    });
}

int mo_attend_backward(const MoAttend* a, void* stream) {
    return guarded([&] {
        if (!attend_sizes(a)) return -1;
        if (a->N == 0) return 0;
        if (a->T && !(rows_usable(a->q, "q", a->dtype) && rows_usable(a->k, "k", a->dtype) && rows_usable(a->v, "v", a->dtype) &&
                      rows_usable(a->dout, "dout", a->dtype) && rows_usable(a->dq, "dq", a->dtype) && rows_usable(a->dk, "dk", a->dtype) &&
                      rows_usable(a->dv, "dv", a->dtype)))
            return -1;
        if (!usable(a->decay, "decay", 4) || (a->state && !usable(a->state, "state", 4)) || (a->T && a->start && !usable(a->start, "start", 1)) ||
            (a->dstate_out && !usable(a->dstate_out, "dstate_out", 4)) || (a->dstate && !usable(a->dstate, "dstate", 4)))
            return -1;
        if (mo_attend_work(a, 1) > 0 && !usable(a->work, "work", 16)) return -1;
        if (a->saved && mo_attend_saved(a) > 0 && !usable(a->saved, "saved", 16)) return -1;
        return by_type(a->dtype, [&](auto t) { return attend_back<decltype(t)>(*a, (hipStream_t)stream); });
    });
}

int mo_attend_step(int dtype, int64_t N, int H, int D, int E, float scale, const MoRows* q, const MoRows* k, const MoRows* v,
                   const float* decay, const uint8_t* start, float* state, const MoRows* out, void* stream) {
    return guarded([&] {
        MoAttend a{};
        a.dtype = dtype; a.T = 1; a.N = N; a.H = H; a.D = D; a.E = E;
        if (!attend_sizes(&a)) return -1;
        if (!q || !k || !v || !out) return fail("invalid arguments (null rows)");
        if (N == 0) return 0;
        if (!rows_usable(*q, "q", dtype) || !rows_usable(*k, "k", dtype) || !rows_usable(*v, "v", dtype) || !rows_usable(*out, "out", dtype) ||
            !usable(decay, "decay", 4) || !usable(state, "state", 4) || (start && !usable(start, "start", 1)))
            return -1;
        const Step st{*q, *k, *v, *out, decay, start, state, N, H, D, E, scale};
        return by_type(dtype, [&](auto t) { return step<decltype(t)>(st, (hipStream_t)stream); });
    });
}

int64_t mo_group_norm_work(const MoNorm* a, int backward) {
    return guarded([&]() -> int64_t {
        if (!norm_sizes(a)) return -1;
        return norm_work(*a, backward != 0);
    });
}

int mo_group_norm(const MoNorm* a, void* stream) {
    return guarded([&] {
        if (!norm_sizes(a)) return -1;
        if (a->B == 0) return 0;
        const size_t z = size_of(a->dtype);
        if (!usable(a->x, "x", z) || !usable(a->y, "y", z) || (a->weight && (!usable(a->weight, "weight", 4) || !usable(a->bias, "bias", 4))) ||
            (a->stats && !usable(a->stats, "stats", 4)) || (norm_work(*a, false) && !usable(a->work, "work", 16)))
            return -1;
        return norm_run(*a, false, (hipStream_t)stream);
    });
}

int mo_group_norm_backward(const MoNorm* a, void* stream) {
    return guarded([&] {
        if (!norm_sizes(a)) return -1;
        if ((!a->dweight) != (!a->dbias)) return fail("dweight and dbias: both or neither");
        if (a->B == 0) return 0;
        const size_t z = size_of(a->dtype);
        if (!usable(a->x, "x", z) || !usable(a->dy, "dy", z) || !usable(a->dx, "dx", z) || !usable(a->stats, "stats", 4) ||
            (a->weight && (!usable(a->weight, "weight", 4) || !usable(a->bias, "bias", 4))) ||
            (a->dweight && (!usable(a->dweight, "dweight", 4) || !usable(a->dbias, "dbias", 4))) ||
            (norm_work(*a, true) && !usable(a->work, "work", 16)))
            return -1;
        return norm_run(*a, true, (hipStream_t)stream);
    });
}

}  // extern "C"
