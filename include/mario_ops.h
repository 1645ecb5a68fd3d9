/* mario_ops: the operators of a policy with a memory, for one AMD MI355X (gfx950) — C ABI of libmario_ops.so.
 *
 * No counterpart in the reference: its policy sees four stacked frames and keeps nothing between steps
 * (ppo/model.py:13-38). These are the operators that a policy needs which remembers the episode: linear attention with a
 * decay for each head, over a stored rollout (with its gradient) and for the single steps of acting, and the group norm with
 * an activation that follows it and the trunk's convolutions; a memory that selects, a state space scan whose decays come from its
 * inputs, with the causal convolution before it, in the same forms; and the norm of all gradients, by which training clips them.
 *
 * Conventions, as in mario_hip.h: plain C types; `stream` is a hipStream_t; every buffer is the caller's memory of the
 * current GPU (device, pinned host or managed), aligned to its elements; functions returning int return 0, or -1 with
 * mo_last_error() (thread-local) set and nothing queued. No call blocks, allocates device memory or keeps anything.
 * Calls are queued on `stream` only, so they may be captured into a graph. */
#ifndef MARIO_OPS_H
#define MARIO_OPS_H
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#pragma GCC visibility push(default)
#endif

/* Last error message of this thread ("" if none). */
const char* mo_last_error(void);

enum { MO_F32 = 0, MO_BF16 = 1 };                       /* element types */
enum { MO_ACT_NONE = 0, MO_ACT_RELU = 1, MO_ACT_SILU = 2 };
#define MO_MAX_HEAD 128                                 /* largest head size */

/* Rows of head vectors: element d of step t, env n, head h at p[t * st + n * sn + h * sh + d] (strides in elements). */
typedef struct MoRows { void* p; int64_t st, sn, sh; } MoRows;

/* Linear attention with a decay for each head. Of env n and head h with g = decay[h]:
 *   S_t = (0 where start[t, n], else g S_{t-1}) + k_t v_t^T,   o_t = scale S_t^T q_t,   S_{-1} = state
 * q, k (T, N, H, D), v, out (T, N, H, E) of one type; sums and states in float32 throughout.
 *   dtype     MO_F32 or MO_BF16;   1 <= D, E <= MO_MAX_HEAD;   T >= 0, N >= 0, H >= 1
 *   decay     (H) float32, each 0 <= g <= 1
 *   start     (T, N) bytes (0, else the step starts an episode: nothing before it is seen), or NULL
 *   state     (N, H, D, E) float32 contiguous, or NULL for zeros
 *   state_out (N, H, D, E) float32: S after the last step; must not overlap state
 *   saved     mo_attend_saved() bytes, 16-byte aligned, for mo_attend_backward to take up, or NULL: no gradient is wanted
 *   work      mo_attend_work() bytes, 16-byte aligned (NULL if 0 are needed), free once the queued work is done
 * For the gradient also: dout (T, N, H, E) and dstate_out (N, H, D, E; NULL: zeros), the gradients of out and state_out, in;
 * dq, dk (T, N, H, D), dv (T, N, H, E) and dstate (N, H, D, E; NULL: not wanted) out; saved as the forward call left it.
 * decay is a constant: there is no gradient for it. Outputs overlap no input. */
typedef struct MoAttend {
    int32_t dtype, H, D, E;
    int64_t T, N;
    float scale;
    MoRows q, k, v, out;
    const float* decay;
    const uint8_t* start;
    const float* state;
    float* state_out;
    void* saved;
    void* work;
    MoRows dout, dq, dk, dv;
    const float* dstate_out;
    float* dstate;
} MoAttend;

/* Bytes of `saved`, and of `work` for the forward (backward = 0) or backward call; sizes and the rows of q, k, v (and dout)
 * have to be set. Heads of whole 16-byte pieces whose rows lie on 16 bytes go by chunks of steps on the matrix cores; others
 * go step by step and need neither. */
int64_t mo_attend_saved(const MoAttend* a);
int64_t mo_attend_work(const MoAttend* a, int backward);
int mo_attend(const MoAttend* a, void* stream);
int mo_attend_backward(const MoAttend* a, void* stream);

/* One step of the same, the state updated in place: q, k, v, out as above with T = 1 (their st is not used), start (N)
 * or NULL, state (N, H, D, E) float32 read and written. A starting env's old state is not read. */
int mo_attend_step(int dtype, int64_t N, int H, int D, int E, float scale, const MoRows* q, const MoRows* k, const MoRows* v,
                   const float* decay, const uint8_t* start, float* state, const MoRows* out, void* stream);

/* Group norm with an activation over channels-last samples: x, y (B, S, C) contiguous (S: a sample's pixels), C channels
 * in `groups` groups of consecutive channels:  y = act(weight (x - mean) rstd + bias), mean and rstd = 1 / sqrt(var + eps)
 * over a sample's S pixels and a group's channels (var the biased one), all in float32.
 *   weight, bias  (C) float32, or both NULL (1 and 0);   act one of MO_ACT_*
 *   stats         (B, groups, 2) float32: mean and rstd out, for the gradient; NULL: not wanted
 *   work          mo_group_norm_work() bytes, 16-byte aligned (NULL if 0), free once the queued work is done
 * The gradient: dy (B, S, C) in, stats from the forward call; dx (B, S, C), dweight and dbias (C; both NULL: not wanted) out.
 * work's size goes by the sizes, by the buffers' alignment and by whether dweight is wanted: set them before asking.
 * The sums over samples and pixels have a fixed order: the same inputs give the same bits. With B = 0 nothing is written. */
typedef struct MoNorm {
    int32_t dtype, act, C, groups;
    int64_t B, S;
    float eps;
    const void* x;
    const float *weight, *bias;
    void* y;
    float* stats;
    void* work;
    const void* dy;
    void* dx;
    float *dweight, *dbias;
} MoNorm;

int64_t mo_group_norm_work(const MoNorm* a, int backward);
int mo_group_norm(const MoNorm* a, void* stream);
int mo_group_norm_backward(const MoNorm* a, void* stream);

/* Causal convolution of each channel over the steps, with an activation. Of env n and channel c, K taps:
 *   y_t = act(bias_c + sum_j weight[c, K - 1 - j] x_{t-j}),  j = 0 .. K - 1, of what the episode of step t holds: terms from before
 * an episode's start are left out, and steps before the first one are the rows of state.
 *   dtype     MO_F32 or MO_BF16 (of x, y, the states and their gradients);   act MO_ACT_*;   C >= 1, 1 <= K <= MO_MAX_TAPS, T, N >= 0
 *   x, y      (T, N, C), channels contiguous; MoRows.sh is not used
 *   weight    (C, K) float32;   bias (C) float32 or NULL
 *   start     (T, N) bytes, as above, or NULL
 *   state     (N, K - 1, C) contiguous: the last K - 1 inputs, oldest first; NULL: zeros
 *   state_out the same after the last step, 0 where its episode holds no input; must not overlap state; NULL: not wanted
 * The gradient: dy (T, N, C) and dstate_out (N, K - 1, C; NULL: zeros) in; dx (T, N, C), dstate (N, K - 1, C; NULL: not wanted), dweight (C, K)
 * and dbias (C) (both NULL: not wanted) out; work mo_conv_work() bytes, 16-byte aligned, free once the queued work is done. Sums are
 * float32 in a fixed order. With N = 0 nothing is written. */
#define MO_MAX_TAPS 8
typedef struct MoConv {
    int32_t dtype, act, C, K;
    int64_t T, N;
    MoRows x, y;
    const float *weight, *bias;
    const uint8_t* start;
    const void* state;
    void* state_out;
    void* work;
    MoRows dy, dx;
    const void* dstate_out;
    void* dstate;
    float *dweight, *dbias;
} MoConv;

int64_t mo_conv_work(const MoConv* a);
int mo_conv(const MoConv* a, void* stream);
int mo_conv_backward(const MoConv* a, void* stream);

/* One step of the same: T is not looked at, x, y (N, C), start (N) or NULL; state_out is read, shifted and written (state is not used). */
int mo_conv_step(const MoConv* a, void* stream);

/* A selective state space scan. Of env n, channel c (in group g of C / G neighbouring ones) and state s:
 *   d_t = softplus(dt_t + dt_bias_c),   h_t = (0 where start[t, n], else exp(d_t A[c, s]) h_{t-1}) + d_t x_t B_t[g, s],
 *   out_t = (sum_s C_t[g, s] h_t + D_c x_t) silu(z_t),   h_{-1} = state
 * States, decays, sums and step sizes d are float32 throughout.
 *   dtype     MO_F32 or MO_BF16 (of x, dt, z, B, C, out and their gradients)
 *   C >= 1, 1 <= S <= MO_MAX_STATES, G >= 1 a divisor of C, T >= 0, N >= 0
 *   x, dt, z, out  (T, N, C), channels contiguous, MoRows.sh not used; z.p NULL: no factor of z
 *   Bt, Ct    (T, N, G, S), states contiguous, MoRows.sh the groups' stride
 *   A         (C, S) float32, none above 0 (a memory that grows may overflow earlier than step by step; an infinite one whose decay over
 *             many steps rounds to 0 becomes NaN);   D, dt_bias (C) float32 or NULL (not there)
 *   start, state, state_out  as for linear attention, states (N, C, S) float32 contiguous
 *   saved     mo_scan_saved() bytes, 16-byte aligned, for mo_scan_backward to take up, or NULL: no gradient is wanted
 *   work      mo_scan_work() bytes, 16-byte aligned, free once the queued work is done
 * The gradient: dout and dstate_out (NULL: zeros) in, saved as the forward call left it; dx, ddt, dz (if z), dB, dC out; dstate (NULL: not
 * wanted) and dA, dD, ddt_bias float32 (each NULL: not wanted) out. Sums have a fixed order: the same inputs give the same bits. With N = 0
 * nothing is written. */
#define MO_MAX_STATES 64
typedef struct MoScan {
    int32_t dtype, C, S, G;
    int64_t T, N;
    MoRows x, dt, z, Bt, Ct, out;
    const float *A, *D, *dt_bias;
    const uint8_t* start;
    const float* state;
    float* state_out;
    void* saved;
    void* work;
    MoRows dout, dx, ddt, dz, dB, dC;
    const float* dstate_out;
    float *dstate, *dA, *dD, *ddt_bias;
} MoScan;

int64_t mo_scan_saved(const MoScan* a);
int64_t mo_scan_work(const MoScan* a, int backward);
int mo_scan(const MoScan* a, void* stream);
int mo_scan_backward(const MoScan* a, void* stream);

/* One step of the same: T is not looked at, x, dt, z, out (N, C), Bt, Ct (N, G, S), start (N) or NULL; state_out (N, C, S) is read and
 * written (state is not used). Nothing of a starting env's old state is seen. */
int mo_scan_step(const MoScan* a, void* stream);

/* The norm of many tensors together, norm = sqrt(sum of all values' squares), and with `scale` their values times
 * min(1, max_norm / (norm + eps)) in place, rounded once. Squares are summed in float64 in a fixed order, so neither large nor tiny
 * values overflow or vanish.
 *   t         count >= 0 tensors in host memory (not needed after the call): n values of a type at p, contiguous; none overlaps another
 *   norm      one float32;   work mo_gradient_work() bytes, 16-byte aligned, free once the queued work is done */
typedef struct MoTensor { void* p; int64_t n; int32_t dtype, reserved; } MoTensor;

int64_t mo_gradient_work(int64_t count);
int mo_gradient_norm(const MoTensor* t, int64_t count, int scale, float max_norm, float eps, float* norm, void* work, void* stream);

#ifdef __cplusplus
#pragma GCC visibility pop
}
#endif
#endif
