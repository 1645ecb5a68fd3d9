// Linear attention one step after another: any head sizes, strides and alignment.
#pragma once
#include "common.hpp"

namespace mo {

// One walk over the steps of an env and head, forwards or backwards in time, with a matrix X that decays:
//   X = (cut ? 0 : g X) + by u_t w_t^T,   y_t = out_by X z_t
// Row a of X belongs to lane a: its B values stay in registers, w_t and z_t come from LDS. Each output of the forward pass
// and of the gradient is such a walk:
//   o:  X = S^T, u = v, w = k, z = q, forwards          dq: X = S,   u = k,  w = v, z = do, forwards
//   dk: X = R,   u = q, w = do, z = v, backwards        dv: X = R^T, u = do, w = q, z = k,  backwards
// with R_t = (start_{t+1} ? 0 : g R_{t+1}) + scale q_t do_t^T the gradient of S_t.
// It takes what the chunk kernels do not: head sizes and strides that are not whole 16-byte pieces, no steps at all, and a gradient
// without what the forward pass saved. Bound by the step after step: a lane's B products and sums wait for LDS reads of w and z that
// all lanes share (128 steps of 1,000 envs, 8 heads of 36, bf16: 855 us, its gradient 2,500).
struct Walk {
    MoRows u, w, z, y;
    const float* decay;
    const uint8_t* start;
    const float* in;           // X before the walk at n * H * A * B + h * A * B + a * sa + b * sb, or null: zeros
    float* out;                // X after it, likewise, or null
    int64_t T, N;
    int H, A, B, sa, sb;
    float by, out_by;
};

constexpr int WALK_STEPS = 16;   // steps whose w and z lie in LDS at a time

template <class T, int BP, bool BACK>
__global__ void __launch_bounds__(kWave) k_walk(Walk k) {
    __shared__ float ws[WALK_STEPS][BP], zs[WALK_STEPS][BP];
    const int64_t nh = block_here(), n = nh / k.H;
    if (n >= k.N) return;
    const int lane = threadIdx.x, h = (int)(nh % k.H), a = blockIdx.y * kWave + lane;
    const bool live = a < k.A;
    const auto at = [&](const MoRows& r, int64_t t) { return (T*)r.p + t * r.st + n * r.sn + h * r.sh; };
    const float g = k.decay[h];
    const int64_t x0 = (n * k.H + h) * (int64_t)k.A * k.B + (int64_t)a * k.sa;
    float X[BP];
#pragma unroll
    for (int b = 0; b < BP; b++) X[b] = live && k.in && b < k.B ? k.in[x0 + (int64_t)b * k.sb] : 0.f;
    for (int64_t s0 = 0; s0 < k.T; s0 += WALK_STEPS) {
        const int steps = (int)(k.T - s0 < WALK_STEPS ? k.T - s0 : WALK_STEPS);
        __syncthreads();
        for (int i = lane; i < steps * k.B; i += kWave) {
            const int j = i / k.B, b = i % k.B;
            const int64_t t = BACK ? k.T - 1 - (s0 + j) : s0 + j;
            ws[j][b] = as_f32(at(k.w, t)[b]);
            zs[j][b] = as_f32(at(k.z, t)[b]);
        }
        __syncthreads();
        for (int j = 0; j < steps; j++) {
            const int64_t t = BACK ? k.T - 1 - (s0 + j) : s0 + j;
            // going back, what decays between t + 1 and t is cut where t + 1 starts an episode; nothing has decayed at the end
            const int64_t ts = BACK ? t + 1 : t;
            const bool cut = k.start && ts < k.T && k.start[ts * k.N + n];
            const float f = BACK && ts == k.T ? 1.f : g;
            const float u = live ? as_f32(at(k.u, t)[a]) * k.by : 0.f;
            float y = 0.f;
#pragma unroll
            for (int b = 0; b < BP; b++)
                if (b < k.B) {
                    X[b] = cut ? u * ws[j][b] : fmaf(f, X[b], u * ws[j][b]);
                    y = fmaf(X[b], zs[j][b], y);
                }
            if (live) at(k.y, t)[a] = as<T>(y * k.out_by);
        }
    }
    if (!live || !k.out) return;
    const bool cut = BACK && k.T && k.start && k.start[n];   // R before the first step: what decays into the entering state
    const float f = BACK && k.T ? g : 1.f;
#pragma unroll
    for (int b = 0; b < BP; b++)
        if (b < k.B) k.out[x0 + (int64_t)b * k.sb] = cut ? 0.f : f * X[b];
}

template <class T, bool BACK> int walk(const Walk& k, hipStream_t s) {
    const dim3 grid = grid_of(k.N * k.H, (k.A + kWave - 1) / kWave);
    if (k.B <= 32) hipLaunchKernelGGL((k_walk<T, 32, BACK>), grid, dim3(kWave), 0, s, k);
    else if (k.B <= 64) hipLaunchKernelGGL((k_walk<T, 64, BACK>), grid, dim3(kWave), 0, s, k);
    else hipLaunchKernelGGL((k_walk<T, 128, BACK>), grid, dim3(kWave), 0, s, k);
    return launched("k_walk");
}

template <class T> int walk_forward(const MoAttend& a, hipStream_t s) {
    return walk<T, false>(Walk{a.v, a.k, a.q, a.out, a.decay, a.start, a.state, a.state_out, a.T, a.N, a.H, a.E, a.D, 1, a.E, 1.f, a.scale}, s);
}

template <class T> int walk_backward(const MoAttend& a, hipStream_t s) {
    if (walk<T, false>(Walk{a.k, a.v, a.dout, a.dq, a.decay, a.start, a.state, nullptr, a.T, a.N, a.H, a.D, a.E, a.E, 1, 1.f, a.scale}, s)) return -1;
    if (walk<T, true>(Walk{a.q, a.dout, a.v, a.dk, a.decay, a.start, a.dstate_out, a.dstate, a.T, a.N, a.H, a.D, a.E, a.E, 1, a.scale, 1.f}, s)) return -1;
    return walk<T, true>(Walk{a.dout, a.q, a.k, a.dv, a.decay, a.start, a.dstate_out, nullptr, a.T, a.N, a.H, a.E, a.D, 1, a.E, a.scale, 1.f}, s);
}

}  // namespace mo
