// libmario_ops.so, second part: the operators of a memory that selects (causal convolution, state space scan) and of the gradients' norm.
#include "conv.hpp"
#include "gradients.hpp"
#include "guard.hpp"
#include "scan.hpp"
#include "scan_back.hpp"
#include "scan_step.hpp"

using namespace mo;

namespace {

bool conv_sizes(const MoConv* a) {
    if (!a || (a->dtype != MO_F32 && a->dtype != MO_BF16) || a->act < MO_ACT_NONE || a->act > MO_ACT_SILU || a->T < 0 || a->N < 0 ||
        a->C < 1 || a->K < 1 || a->K > MO_MAX_TAPS) {
        fail("invalid arguments (dtype MO_F32 or MO_BF16, act MO_ACT_*, T >= 0, N >= 0, C >= 1, K 1 .. 8)");
        return false;
    }
    if (a->C > (1 << 20) || a->N >= MAX_GRID || a->T > ((int64_t)1 << 40)) { fail("too many channels, envs or steps (C <= 2^20, N < 2^31, T <= 2^40)"); return false; }
    if ((!a->dweight) != (!a->dbias)) { fail("dweight and dbias: both or neither"); return false; }
    return true;
}
bool conv_params(const MoConv* a) { return usable(a->weight, "weight", 4) && (!a->bias || usable(a->bias, "bias", 4)); }
bool maybe(const void* p, const char* name, size_t align) { return !p || usable(p, name, align); }

template <class T, int RUN> int conv_run(const MoConv& a, hipStream_t s) {
    return by_act(a.act, [&](auto act) {
        constexpr int A = decltype(act)::value;
        const int V = conv_width(a, RUN == 1, RUN == 2);
        if constexpr (sizeof(T) == 2) {
            if (V == 8) return conv_taps<T, 8, RUN, A, 1, RUN == 1 ? 4 : MO_MAX_TAPS>(a, s);
            if constexpr (RUN == 1)
                if (V == 4) return conv_taps<T, 4, RUN, A, 5>(a, s);
        } else {
            if (V == 4) return conv_taps<T, 4, RUN, A>(a, s);
        }
        return conv_taps<T, 1, RUN, A>(a, s);
    });
}

bool scan_sizes(const MoScan* a) {
    if (!a || (a->dtype != MO_F32 && a->dtype != MO_BF16) || a->T < 0 || a->N < 0 || a->C < 1 || a->S < 1 || a->S > MO_MAX_STATES ||
        a->G < 1 || a->C % a->G) {
        fail("invalid arguments (dtype MO_F32 or MO_BF16, T >= 0, N >= 0, C a multiple of G >= 1, S 1 .. 64)");
        return false;
    }
    if (a->C > (1 << 20) || a->N >= MAX_GRID || a->T > ((int64_t)1 << 40)) { fail("too many channels, envs or steps (C <= 2^20, N < 2^31, T <= 2^40)"); return false; }
    return true;
}
bool scan_params(const MoScan* a) { return usable(a->A, "A", 4) && maybe(a->D, "D", 4) && maybe(a->dt_bias, "dt_bias", 4); }
bool scan_rows(const MoScan* a) {
    const size_t z = size_of(a->dtype);
    return usable(a->x.p, "x", z) && usable(a->dt.p, "dt", z) && maybe(a->z.p, "z", z) && usable(a->Bt.p, "Bt", z) && usable(a->Ct.p, "Ct", z);
}

}  // namespace

extern "C" {

int64_t mo_conv_work(const MoConv* a) {
    return guarded([&]() -> int64_t { return conv_sizes(a) ? conv_back_work(*a) : -1; });
}

int mo_conv(const MoConv* a, void* stream) {
    return guarded([&] {
        if (!conv_sizes(a)) return -1;
        if (a->N == 0) return 0;
        const size_t z = size_of(a->dtype);
        if (!conv_params(a) || (a->T && !(usable(a->x.p, "x", z) && usable(a->y.p, "y", z) && maybe(a->start, "start", 1))) ||
            (a->K > 1 && !(maybe(a->state, "state", z) && maybe(a->state_out, "state_out", z))))
            return -1;
        return by_type(a->dtype, [&](auto t) { return conv_run<decltype(t), 0>(*a, (hipStream_t)stream); });
    });
}

int mo_conv_backward(const MoConv* a, void* stream) {
    return guarded([&] {
        if (!conv_sizes(a)) return -1;
        if (a->N == 0) return 0;
        const size_t z = size_of(a->dtype);
        if (!conv_params(a) || (a->T && !(usable(a->x.p, "x", z) && usable(a->dy.p, "dy", z) && usable(a->dx.p, "dx", z) && maybe(a->start, "start", 1))) ||
            (a->K > 1 && !(maybe(a->state, "state", z) && maybe(a->dstate_out, "dstate_out", z) && maybe(a->dstate, "dstate", z))) ||
            (a->dweight && !(usable(a->dweight, "dweight", 4) && usable(a->dbias, "dbias", 4))) || (conv_back_work(*a) && !usable(a->work, "work", 16)))
            return -1;
        return by_type(a->dtype, [&](auto t) { return conv_run<decltype(t), 1>(*a, (hipStream_t)stream); });
    });
}

int mo_conv_step(const MoConv* a, void* stream) {
    return guarded([&] {
        if (!conv_sizes(a)) return -1;
        if (a->N == 0) return 0;
        const size_t z = size_of(a->dtype);
        if (!conv_params(a) || !usable(a->x.p, "x", z) || !usable(a->y.p, "y", z) || !maybe(a->start, "start", 1) ||
            (a->K > 1 && !usable(a->state_out, "state_out", z)))
            return -1;
        return by_type(a->dtype, [&](auto t) { return conv_run<decltype(t), 2>(*a, (hipStream_t)stream); });
    });
}

int64_t mo_scan_saved(const MoScan* a) {
    return guarded([&]() -> int64_t {
        if (!scan_sizes(a)) return -1;
        const Scan k = scan_cut(*a, false);
        return 4 * (scan_bc(k) + scan_kept(k));
    });
}

int64_t mo_scan_work(const MoScan* a, int backward) {
    return guarded([&]() -> int64_t { return scan_sizes(a) ? 4 * scan_work_floats(scan_cut(*a, backward), backward) : -1; });
}

int mo_scan(const MoScan* a, void* stream) {
    return guarded([&] {
        if (!scan_sizes(a)) return -1;
        if (a->N == 0) return 0;
        if (!scan_params(a) || (a->T && !(scan_rows(a) && usable(a->out.p, "out", size_of(a->dtype)) && maybe(a->start, "start", 1))) ||
            !maybe(a->state, "state", 4) || !usable(a->state_out, "state_out", 4) || (mo_scan_work(a, 0) && !usable(a->work, "work", 16)) ||
            (a->saved && mo_scan_saved(a) && !usable(a->saved, "saved", 16)))
            return -1;
        return by_type(a->dtype, [&](auto t) { return scan_forward<decltype(t)>(*a, (hipStream_t)stream); });
    });
}

int mo_scan_backward(const MoScan* a, void* stream) {
    return guarded([&] {
        if (!scan_sizes(a)) return -1;
        if (a->N == 0) return 0;
        const size_t z = size_of(a->dtype);
        if (!scan_params(a) ||
            (a->T && !(scan_rows(a) && usable(a->dout.p, "dout", z) && usable(a->dx.p, "dx", z) && usable(a->ddt.p, "ddt", z) &&
                       (!a->z.p || usable(a->dz.p, "dz", z)) && usable(a->dB.p, "dB", z) && usable(a->dC.p, "dC", z) && maybe(a->start, "start", 1) &&
                       usable(a->saved, "saved", 16))) ||
            !maybe(a->dstate_out, "dstate_out", 4) || !maybe(a->dstate, "dstate", 4) || !maybe(a->dA, "dA", 4) || !maybe(a->dD, "dD", 4) ||
            !maybe(a->ddt_bias, "ddt_bias", 4) || (mo_scan_work(a, 1) && !usable(a->work, "work", 16)))
            return -1;
        return by_type(a->dtype, [&](auto t) { return scan_backward<decltype(t)>(*a, (hipStream_t)stream); });
    });
}

int mo_scan_step(const MoScan* a, void* stream) {
    return guarded([&] {
        if (!scan_sizes(a)) return -1;
        if (a->N == 0) return 0;
        if (!scan_params(a) || !scan_rows(a) || !usable(a->out.p, "out", size_of(a->dtype)) || !maybe(a->start, "start", 1) || !usable(a->state_out, "state_out", 4))
            return -1;
        return by_type(a->dtype, [&](auto t) { return scan_step<decltype(t)>(*a, (hipStream_t)stream); });
    });
}

int64_t mo_gradient_work(int64_t count) {
    if (count < 0) return fail("invalid arguments (count >= 0)");
    return gradient_work(count);
}

int mo_gradient_norm(const MoTensor* t, int64_t count, int scale, float max_norm, float eps, float* norm, void* work, void* stream) {
    return guarded([&] {
        if (count < 0 || (count && !t) || (scale && !(max_norm >= 0.f && eps >= 0.f))) return fail("invalid arguments (count >= 0 tensors, max_norm >= 0, eps >= 0)");
        int64_t chunks = 0;
        for (int64_t i = 0; i < count; i++) {
            if ((t[i].dtype != MO_F32 && t[i].dtype != MO_BF16) || t[i].n < 0 || t[i].n > ((int64_t)1 << 44)) return fail("tensors: MO_F32 or MO_BF16, 0 .. 2^44 values");
            if (t[i].n && !usable(t[i].p, "tensor", size_of(t[i].dtype))) return -1;
            chunks += (t[i].n + GRADIENT_CHUNK - 1) / GRADIENT_CHUNK;
        }
        if (chunks >= ((int64_t)1 << 32)) return fail("tensors: too many values");
        if (!usable(norm, "norm", 4) || !usable(work, "work", 16)) return -1;
        return gradient_norm(t, count, scale != 0, max_norm, eps, norm, (double*)work, (hipStream_t)stream);
    });
}

}  // extern "C"
