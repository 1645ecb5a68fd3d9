// The operators of libmario_ops.so on torch tensors: allocation, views, streams and autograd. Their host work is most of a small
// call's time, and in a training step it runs on autograd's own thread, so none of it is left to Python. Arguments come checked
// (memory.py): plain tensors of one GPU with the types and shapes that include/mario_ops.h asks for.
#include <ATen/ATen.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/utils/pybind.h>

#include <algorithm>
#include <optional>
#include <string>
#include <vector>

#include "../../../include/mario_ops.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

int64_t ok(int64_t rc, const char* what) {
    TORCH_CHECK(rc >= 0, what, " failed: ", mo_last_error());
    return rc;
}
void* stream_of(const Tensor& t) { return c10::hip::getCurrentHIPStream(t.device().index()).stream(); }
int dtype_of(const Tensor& t) { return t.scalar_type() == at::kBFloat16 ? MO_BF16 : MO_F32; }
template <class T = float> T* data(const Tensor& t) { return t.defined() ? (T*)t.data_ptr() : nullptr; }

Tensor work_of(int64_t bytes, const Tensor& like) {
    return bytes ? at::empty({bytes}, like.options().dtype(at::kByte)) : Tensor();
}

// Head vectors (T, N, H, d) or (N, H, d), the last dimension contiguous.
MoRows rows_of(const Tensor& t) {
    const auto st = t.strides();
    return t.dim() == 4 ? MoRows{t.data_ptr(), st[0], st[1], st[2]} : MoRows{t.data_ptr(), 0, st[0], st[1]};
}
// The tensor as the kernels take it: head vectors contiguous, and on 16-byte boundaries where their size allows it (they are copied
// otherwise: a copy costs less than going step by step).
Tensor as_rows(const Tensor& t) {
    const auto st = t.strides();
    const int64_t d = t.size(-1), whole = 16 / t.element_size();
    if (st.back() != 1 && d != 1) return t.contiguous();
    if (d % whole) return t;
    bool suits = (uintptr_t)t.data_ptr() % 16 == 0;
    for (size_t i = 0; i + 1 < st.size(); i++) suits = suits && st[i] % whole == 0;
    return suits ? t : t.clone(at::MemoryFormat::Contiguous);
}
Tensor contiguous(const Tensor& t) { return t.defined() ? t.contiguous() : t; }
typedef std::optional<Tensor> Maybe;   // (autograd takes no undefined tensors as inputs)
Maybe maybe(const Tensor& t) { return t.defined() ? Maybe(t) : std::nullopt; }
Tensor sure(const Maybe& t) { return t ? *t : Tensor(); }

bool wants_grad(at::ArrayRef<Tensor> ts) {
    if (!at::GradMode::is_enabled()) return false;
    for (const Tensor& t : ts)
        if (t.defined() && t.requires_grad()) return true;
    return false;
}
void written(const Tensor& t) {
    if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();   // (what saved it for a gradient notices)
}
// Gradients of a pass that has no gradient itself: where one is asked for all the same, an error.
variable_list once(variable_list grads) {
    if (!at::GradMode::is_enabled()) return grads;
    variable_list in;
    for (Tensor& g : grads)
        if (g.defined()) in.push_back(g.detach().set_requires_grad(true));
    auto error = std::make_shared<torch::autograd::DelayedError>("this operator is differentiable once", (int64_t)in.size());
    variable_list out = (*error)(std::move(in));
    size_t i = 0;
    for (Tensor& g : grads)
        if (g.defined()) g = out[i++];
    return grads;
}

// ---------------------------------------------------------------- linear attention
MoAttend attend_args(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& decay, const Tensor& start, const Tensor& state, double scale) {
    MoAttend a{};
    a.dtype = dtype_of(q);
    a.T = q.size(0); a.N = q.size(1); a.H = (int32_t)q.size(2); a.D = (int32_t)q.size(3); a.E = (int32_t)v.size(3);
    a.scale = (float)scale;
    a.q = rows_of(q); a.k = rows_of(k); a.v = rows_of(v);
    a.decay = data(decay);
    a.start = data<uint8_t>(start);
    a.state = data(state);
    return a;
}

struct Forward { Tensor out, state, saved; };
Forward attend_forward(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& decay, const Tensor& start, const Tensor& state, double scale, bool keep) {
    const c10::DeviceGuard guard(q.device());
    MoAttend a = attend_args(q, k, v, decay, start, state, scale);
    Forward f;
    f.out = at::empty({a.T, a.N, a.H, a.E}, q.options());
    f.state = at::empty({a.N, a.H, a.D, a.E}, q.options().dtype(at::kFloat));
    a.out = rows_of(f.out);
    a.state_out = data(f.state);
    if (keep) f.saved = work_of(ok(mo_attend_saved(&a), "mo_attend_saved"), q);
    const Tensor work = work_of(ok(mo_attend_work(&a, 0), "mo_attend_work"), q);
    a.saved = data<void>(f.saved);
    a.work = data<void>(work);
    ok(mo_attend(&a, stream_of(q)), "mo_attend");
    return f;
}

struct Attend : torch::autograd::Function<Attend> {
    static variable_list forward(AutogradContext* ctx, Tensor q, Tensor k, Tensor v, Tensor decay, Maybe start_, Maybe state_, double scale) {
        const Tensor start = sure(start_), state = sure(state_);
        Forward f = attend_forward(q, k, v, decay, start, state, scale, true);
        ctx->save_for_backward({q, k, v, decay, start, state, f.saved});
        ctx->saved_data["scale"] = scale;
        ctx->saved_data["state"] = (int64_t)(start.defined() ? 5 : 4);   // its place among the tensors
        ctx->set_materialize_grads(false);
        return {f.out, f.state};
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        const variable_list s = ctx->get_saved_variables();
        const Tensor &q = s[0], &k = s[1], &v = s[2], &state = s[5];
        const c10::DeviceGuard guard(q.device());
        MoAttend a = attend_args(q, k, v, s[3], s[4], state, ctx->saved_data["scale"].toDouble());
        const Tensor dout = as_rows(grads[0].defined() ? grads[0] : at::zeros({1}, q.options()).expand(v.sizes()));
        const Tensor dstate_out = contiguous(grads[1]);
        const Tensor dq = at::empty(q.sizes(), q.options()), dk = at::empty(k.sizes(), q.options()), dv = at::empty(v.sizes(), q.options());
        const Tensor dstate = state.defined() && ctx->needs_input_grad((size_t)ctx->saved_data["state"].toInt()) ? at::empty(state.sizes(), state.options()) : Tensor();
        a.saved = data<void>(s[6]);
        a.dout = rows_of(dout); a.dq = rows_of(dq); a.dk = rows_of(dk); a.dv = rows_of(dv);
        a.dstate_out = data(dstate_out);
        a.dstate = data(dstate);
        const Tensor work = work_of(ok(mo_attend_work(&a, 1), "mo_attend_work"), q);
        a.work = data<void>(work);
        ok(mo_attend_backward(&a, stream_of(q)), "mo_attend_backward");
        return once({dq, dk, dv, Tensor(), Tensor(), dstate, Tensor()});
    }
};

std::tuple<Tensor, Tensor> attend(const Tensor& q_, const Tensor& k_, const Tensor& v_, const Tensor& decay_, const Maybe& start_,
                                  const Maybe& state_, double scale) {
    const Tensor q = as_rows(q_), k = as_rows(k_), v = as_rows(v_), decay = decay_.contiguous();
    const Tensor start = contiguous(sure(start_)), state = contiguous(sure(state_));
    if (wants_grad({q, k, v, state})) {
        const variable_list out = Attend::apply(q, k, v, decay, maybe(start), maybe(state), scale);
        return {out[0], out[1]};
    }
    const Forward f = attend_forward(q, k, v, decay, start, state, scale, false);
    return {f.out, f.state};
}

Tensor attend_step(const Tensor& q_, const Tensor& k_, const Tensor& v_, const Tensor& decay_, const Tensor& state, const Maybe& start_, double scale) {
    const c10::DeviceGuard guard(q_.device());
    const Tensor q = as_rows(q_), k = as_rows(k_), v = as_rows(v_), decay = decay_.contiguous(), start = contiguous(sure(start_));
    const Tensor out = at::empty(v.sizes(), v.options());
    const MoRows rq = rows_of(q), rk = rows_of(k), rv = rows_of(v), ro = rows_of(out);
    ok(mo_attend_step(dtype_of(q), q.size(0), (int)q.size(1), (int)q.size(2), (int)v.size(2), (float)scale, &rq, &rk, &rv, data(decay),
                      data<uint8_t>(start), data(state), &ro, stream_of(q)),
       "mo_attend_step");
    written(state);
    return out;
}

// ---------------------------------------------------------------- group norm and activation
// x (B, C, ...) as its channels-last rows (B, ..., C), contiguous (a copy where it lies otherwise), and back.
Tensor channels_last(const Tensor& x) { return (x.dim() > 2 ? x.movedim(1, -1) : x).contiguous(); }
Tensor channels_second(const Tensor& rows) { return rows.dim() > 2 ? rows.movedim(-1, 1) : rows; }

MoNorm norm_args(const Tensor& rows, int64_t groups, const Tensor& weight, const Tensor& bias, double eps, int64_t act) {
    MoNorm a{};
    a.dtype = dtype_of(rows);
    a.act = (int32_t)act;
    a.B = rows.size(0);
    a.C = (int32_t)rows.size(-1);
    a.S = a.B ? rows.numel() / (a.B * a.C) : 1;
    a.groups = (int32_t)groups;
    a.eps = (float)eps;
    a.x = rows.data_ptr();
    a.weight = data(weight);
    a.bias = data(bias);
    return a;
}

// The result has the channels second and rows' memory order without being a view of another tensor: a view that an autograd
// function returns may not be changed in place.
Tensor norm_forward(const Tensor& rows, int64_t groups, const Tensor& weight, const Tensor& bias, double eps, int64_t act, Tensor* stats) {
    const c10::DeviceGuard guard(rows.device());
    MoNorm a = norm_args(rows, groups, weight, bias, eps, act);
    const Tensor second = channels_second(rows), y = at::empty_strided(second.sizes(), second.strides(), rows.options());
    if (stats) *stats = at::empty({a.B, groups, 2}, rows.options().dtype(at::kFloat));
    a.y = y.data_ptr();
    a.stats = stats ? data(*stats) : nullptr;
    const Tensor work = work_of(ok(mo_group_norm_work(&a, 0), "mo_group_norm_work"), rows);
    a.work = data<void>(work);
    ok(mo_group_norm(&a, stream_of(rows)), "mo_group_norm");
    return y;
}

struct Norm : torch::autograd::Function<Norm> {
    static Tensor forward(AutogradContext* ctx, Tensor x, int64_t groups, Maybe weight_, Maybe bias_, double eps, int64_t act) {
        const Tensor weight = sure(weight_), bias = sure(bias_);
        const Tensor rows = channels_last(x);
        Tensor stats;
        const Tensor y = norm_forward(rows, groups, weight, bias, eps, act, &stats);
        ctx->save_for_backward({rows, weight, bias, stats});
        ctx->saved_data["groups"] = groups;
        ctx->saved_data["eps"] = eps;
        ctx->saved_data["act"] = act;
        return y;
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        const variable_list s = ctx->get_saved_variables();
        const Tensor &rows = s[0], &weight = s[1], dy = channels_last(grads[0]), dx = at::empty_like(rows);
        const c10::DeviceGuard guard(rows.device());
        MoNorm a = norm_args(rows, ctx->saved_data["groups"].toInt(), weight, s[2], ctx->saved_data["eps"].toDouble(), ctx->saved_data["act"].toInt());
        Tensor dw, db;
        if (weight.defined() && (ctx->needs_input_grad(1) || ctx->needs_input_grad(2))) {
            const Tensor both = a.B ? at::empty({2, a.C}, weight.options()) : at::zeros({2, a.C}, weight.options());
            dw = both.select(0, 0);
            db = both.select(0, 1);
        }
        a.stats = data(s[3]);
        a.dy = dy.data_ptr();
        a.dx = dx.data_ptr();
        a.dweight = data(dw);
        a.dbias = data(db);
        const Tensor work = work_of(ok(mo_group_norm_work(&a, 1), "mo_group_norm_work"), rows);
        a.work = data<void>(work);
        ok(mo_group_norm_backward(&a, stream_of(rows)), "mo_group_norm_backward");
        return once({channels_second(dx), Tensor(), dw, db, Tensor(), Tensor()});
    }
};

Tensor group_norm_act(const Tensor& x, int64_t groups, const Maybe& weight_, const Maybe& bias_, double eps, int64_t act) {
    Tensor weight, bias;
    if (weight_) {
        weight = weight_->to(at::kFloat).contiguous();
        bias = bias_->to(at::kFloat).contiguous();
    }
    if (wants_grad({x, weight, bias})) return Norm::apply(x, groups, maybe(weight), maybe(bias), eps, act);
    return norm_forward(channels_last(x), groups, weight, bias, eps, act, nullptr);
}

// ---------------------------------------------------------------- causal convolution and activation
// Values of channels (T, N, C) or (N, C), the channels contiguous.
MoRows channel_rows(const Tensor& t) {
    if (!t.defined()) return MoRows{};
    const auto st = t.strides();
    return t.dim() == 3 ? MoRows{t.data_ptr(), st[0], st[1], 0} : MoRows{t.data_ptr(), 0, st[0], 0};
}
// As the scan's kernels take them: contiguous along the last dimension.
Tensor inner(const Tensor& t) { return !t.defined() || t.strides().back() == 1 || t.size(-1) == 1 ? t : t.contiguous(); }
Tensor float_param(const Maybe& t) { return t ? t->to(at::kFloat).contiguous() : Tensor(); }

MoConv conv_args(const Tensor& x, const Tensor& weight, const Tensor& bias, const Tensor& start, const Tensor& state, int64_t act) {
    MoConv a{};
    a.dtype = dtype_of(x);
    a.act = (int32_t)act;
    a.T = x.dim() == 3 ? x.size(0) : 1; a.N = x.size(-2); a.C = (int32_t)x.size(-1); a.K = (int32_t)weight.size(1);
    a.x = channel_rows(x);
    a.weight = data(weight);
    a.bias = data(bias);
    a.start = data<uint8_t>(start);
    a.state = data<void>(state);
    return a;
}
std::pair<Tensor, Tensor> conv_forward(const Tensor& x, const Tensor& weight, const Tensor& bias, const Tensor& start, const Tensor& state, int64_t act) {
    const c10::DeviceGuard guard(x.device());
    MoConv a = conv_args(x, weight, bias, start, state, act);
    const Tensor y = at::empty(x.sizes(), x.options()), last = at::empty({a.N, a.K - 1, a.C}, x.options());
    a.y = channel_rows(y);
    a.state_out = data<void>(last);
    ok(mo_conv(&a, stream_of(x)), "mo_conv");
    return {y, last};
}

struct Conv : torch::autograd::Function<Conv> {
    static variable_list forward(AutogradContext* ctx, Tensor x, Tensor weight, Maybe bias_, Maybe start_, Maybe state_, int64_t act) {
        const Tensor bias = sure(bias_), start = sure(start_), state = sure(state_);
        const auto [y, last] = conv_forward(x, weight, bias, start, state, act);
        ctx->save_for_backward({x, weight, bias, start, state});
        ctx->saved_data["act"] = act;
        ctx->set_materialize_grads(false);
        return {y, last};
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        const variable_list s = ctx->get_saved_variables();
        const Tensor &x = s[0], &weight = s[1], &bias = s[2], &start = s[3], &state = s[4];
        const c10::DeviceGuard guard(x.device());
        MoConv a = conv_args(x, weight, bias, start, state, ctx->saved_data["act"].toInt());
        const Tensor dy = as_rows(grads[0].defined() ? grads[0] : at::zeros({1}, x.options()).expand(x.sizes()));
        const Tensor dlast = contiguous(grads[1]), dx = at::empty(x.sizes(), x.options());
        // inputs that are there, in their order: x, weight, bias, start, state
        size_t at = 1;
        const bool want_weight = ctx->needs_input_grad(at);
        const bool want_bias = bias.defined() && ctx->needs_input_grad(++at);
        if (start.defined()) ++at;
        const Tensor dstate = state.defined() && ctx->needs_input_grad(++at) ? at::empty(state.sizes(), state.options()) : Tensor();
        Tensor dw, db;
        if (want_weight || want_bias) {
            const auto make = [&](at::IntArrayRef size) { return a.N && a.T ? at::empty(size, weight.options()) : at::zeros(size, weight.options()); };
            dw = make(weight.sizes());
            db = make({a.C});
        }
        a.dy = channel_rows(dy);
        a.dx = channel_rows(dx);
        a.dstate_out = data<void>(dlast);
        a.dstate = data<void>(dstate);
        a.dweight = data(dw);
        a.dbias = data(db);
        const Tensor work = work_of(ok(mo_conv_work(&a), "mo_conv_work"), x);
        a.work = data<void>(work);
        ok(mo_conv_backward(&a, stream_of(x)), "mo_conv_backward");
        return once({dx, dw, bias.defined() ? db : Tensor(), Tensor(), dstate, Tensor()});
    }
};

std::tuple<Tensor, Tensor> conv(const Tensor& x_, const Tensor& weight_, const Maybe& bias_, const Maybe& start_, const Maybe& state_, int64_t act) {
    const Tensor x = as_rows(x_), weight = weight_.to(at::kFloat).contiguous(), bias = float_param(bias_);
    const Tensor start = contiguous(sure(start_)), state = contiguous(sure(state_));
    if (wants_grad({x, weight, bias, state})) {
        const variable_list out = Conv::apply(x, weight, maybe(bias), maybe(start), maybe(state), act);
        return {out[0], out[1]};
    }
    const auto [y, last] = conv_forward(x, weight, bias, start, state, act);
    return {y, last};
}

Tensor conv_step(const Tensor& x_, const Tensor& weight_, const Maybe& bias_, const Tensor& state, const Maybe& start_, int64_t act) {
    const c10::DeviceGuard guard(x_.device());
    const Tensor x = as_rows(x_), weight = weight_.to(at::kFloat).contiguous(), bias = float_param(bias_), start = contiguous(sure(start_));
    MoConv a = conv_args(x, weight, bias, start, Tensor(), act);
    const Tensor y = at::empty(x.sizes(), x.options());
    a.y = channel_rows(y);
    a.state_out = data<void>(state);
    ok(mo_conv_step(&a, stream_of(x)), "mo_conv_step");
    written(state);
    return y;
}

// ---------------------------------------------------------------- selective state space scan
struct ScanIn { Tensor x, dt, A, B, C, D, z, bias, start, state; };
MoScan scan_args(const ScanIn& in) {
    MoScan a{};
    a.dtype = dtype_of(in.x);
    a.T = in.x.dim() == 3 ? in.x.size(0) : 1; a.N = in.x.size(-2); a.C = (int32_t)in.x.size(-1);
    a.S = (int32_t)in.A.size(1); a.G = (int32_t)in.B.size(-2);
    a.x = channel_rows(in.x); a.dt = channel_rows(in.dt); a.z = channel_rows(in.z);
    a.Bt = rows_of(in.B); a.Ct = rows_of(in.C);
    a.A = data(in.A); a.D = data(in.D); a.dt_bias = data(in.bias);
    a.start = data<uint8_t>(in.start);
    a.state = data(in.state);
    return a;
}
Forward scan_forward(const ScanIn& in, bool keep) {
    const c10::DeviceGuard guard(in.x.device());
    MoScan a = scan_args(in);
    Forward f;
    f.out = at::empty(in.x.sizes(), in.x.options());
    f.state = at::empty({a.N, a.C, a.S}, in.x.options().dtype(at::kFloat));
    a.out = channel_rows(f.out);
    a.state_out = data(f.state);
    if (keep) f.saved = work_of(ok(mo_scan_saved(&a), "mo_scan_saved"), in.x);
    a.saved = data<void>(f.saved);
    const Tensor work = work_of(ok(mo_scan_work(&a, 0), "mo_scan_work"), in.x);
    a.work = data<void>(work);
    ok(mo_scan(&a, stream_of(in.x)), "mo_scan");
    return f;
}

struct StateScan : torch::autograd::Function<StateScan> {
    static variable_list forward(AutogradContext* ctx, Tensor x, Tensor dt, Tensor A, Tensor B, Tensor C, Maybe D, Maybe z, Maybe bias, Maybe start, Maybe state) {
        const ScanIn in{x, dt, A, B, C, sure(D), sure(z), sure(bias), sure(start), sure(state)};
        Forward f = scan_forward(in, true);
        ctx->save_for_backward({x, dt, A, B, C, in.D, in.z, in.bias, in.start, in.state, f.saved});
        ctx->set_materialize_grads(false);
        return {f.out, f.state};
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        const variable_list s = ctx->get_saved_variables();
        const ScanIn in{s[0], s[1], s[2], s[3], s[4], s[5], s[6], s[7], s[8], s[9]};
        const c10::DeviceGuard guard(in.x.device());
        MoScan a = scan_args(in);
        const Tensor dout = inner(grads[0].defined() ? grads[0] : at::zeros({1}, in.x.options()).expand(in.x.sizes()));
        const Tensor dlast = contiguous(grads[1]);
        // inputs that are there, in their order
        size_t at = 5;
        const auto wants = [&](const Tensor& t) { return t.defined() && ctx->needs_input_grad(at++); };
        const bool want_D = wants(in.D);
        wants(in.z);
        const bool want_bias = wants(in.bias);
        wants(in.start);
        const bool want_state = wants(in.state);
        const auto like = [](const Tensor& t) { return at::empty(t.sizes(), t.options()); };
        const auto sums = [&](bool want, const Tensor& t) { return !want ? Tensor() : a.N && a.T ? like(t) : at::zeros(t.sizes(), t.options()); };
        const Tensor dx = like(in.x), ddt = like(in.dt), dB = like(in.B), dC = like(in.C), dz = in.z.defined() ? like(in.z) : Tensor();
        const Tensor dA = sums(ctx->needs_input_grad(2), in.A), dD = sums(want_D, in.D), dbias = sums(want_bias, in.bias);
        const Tensor dstate = want_state ? like(in.state) : Tensor();
        a.saved = data<void>(s[10]);
        a.dout = channel_rows(dout); a.dx = channel_rows(dx); a.ddt = channel_rows(ddt); a.dz = channel_rows(dz);
        a.dB = rows_of(dB); a.dC = rows_of(dC);
        a.dstate_out = data(dlast);
        a.dstate = data(dstate); a.dA = data(dA); a.dD = data(dD); a.ddt_bias = data(dbias);
        const Tensor work = work_of(ok(mo_scan_work(&a, 1), "mo_scan_work"), in.x);
        a.work = data<void>(work);
        ok(mo_scan_backward(&a, stream_of(in.x)), "mo_scan_backward");
        return once({dx, ddt, dA, dB, dC, dD, dz, dbias, Tensor(), dstate});
    }
};

ScanIn scan_in(const Tensor& x, const Tensor& dt, const Tensor& A, const Tensor& B, const Tensor& C, const Maybe& D, const Maybe& z, const Maybe& bias,
               const Maybe& start, const Maybe& state) {
    return {inner(x), inner(dt), A.to(at::kFloat).contiguous(), inner(B), inner(C), float_param(D), inner(sure(z)), float_param(bias),
            contiguous(sure(start)), contiguous(sure(state))};
}
std::tuple<Tensor, Tensor> scan(const Tensor& x, const Tensor& dt, const Tensor& A, const Tensor& B, const Tensor& C, const Maybe& D, const Maybe& z,
                                const Maybe& bias, const Maybe& start, const Maybe& state) {
    const ScanIn in = scan_in(x, dt, A, B, C, D, z, bias, start, state);
    if (wants_grad({in.x, in.dt, in.A, in.B, in.C, in.D, in.z, in.bias, in.state})) {
        const variable_list out = StateScan::apply(in.x, in.dt, in.A, in.B, in.C, maybe(in.D), maybe(in.z), maybe(in.bias), maybe(in.start), maybe(in.state));
        return {out[0], out[1]};
    }
    const Forward f = scan_forward(in, false);
    return {f.out, f.state};
}

Tensor scan_step(const Tensor& x, const Tensor& dt, const Tensor& A, const Tensor& B, const Tensor& C, const Tensor& state, const Maybe& D, const Maybe& z,
                 const Maybe& bias, const Maybe& start) {
    const c10::DeviceGuard guard(x.device());
    const ScanIn in = scan_in(x, dt, A, B, C, D, z, bias, start, std::nullopt);
    MoScan a = scan_args(in);
    const Tensor out = at::empty(x.sizes(), x.options());
    a.out = channel_rows(out);
    a.state_out = data(state);
    ok(mo_scan_step(&a, stream_of(x)), "mo_scan_step");
    written(state);
    return out;
}

// ---------------------------------------------------------------- the gradients' norm
// Tensors that fill their memory without gaps are taken as they lie; others by a copy, which goes back after scaling. None where they are to be
// scaled and the spans of two cross, unless the caller knows them `apart`: whether they share elements takes longer to find out.
Maybe gradient_norm(const std::string& name, const std::vector<Tensor>& given, bool scale, double max_norm, double eps, bool apart) {
    const Tensor& first = given[0];
    const c10::DeviceGuard guard(first.device());
    const at::NoGradGuard no_grad;
    const auto lies = [](const Tensor& g) { return g.is_non_overlapping_and_dense() && !g.is_neg(); };
    std::vector<std::pair<char*, char*>> spans;
    spans.reserve(given.size());
    for (const Tensor& g : given) {
        TORCH_CHECK_VALUE(g.layout() == at::kStrided && g.is_floating_point() && g.device() == first.device(), name, ": gradients must be dense float tensors on one device");
        TORCH_CHECK_VALUE(g.scalar_type() == at::kFloat || g.scalar_type() == at::kBFloat16, name, ": gradients on the GPU must be float32 or bf16");
        const bool as_it_lies = lies(g);
        int64_t last = 0;
        for (int64_t d = 0; d < g.dim() && !as_it_lies; d++) {
            TORCH_CHECK_VALUE(g.stride(d) || g.size(d) < 2, name, ": a gradient shares elements with itself (expanded)");
            last += (g.size(d) - 1) * g.stride(d);
        }
        char* const at = (char*)g.data_ptr();
        if (scale && !apart && g.numel()) spans.push_back({at, at + (as_it_lies ? g.numel() : last + 1) * g.element_size()});
    }
    std::sort(spans.begin(), spans.end());
    for (size_t i = 1; i < spans.size(); i++)
        if (spans[i].first < spans[i - 1].second) return std::nullopt;
    std::vector<Tensor> held;
    std::vector<MoTensor> list;
    held.reserve(given.size());
    list.reserve(given.size());
    for (const Tensor& g : given) {
        held.push_back(lies(g) ? g : g.is_neg() ? g.resolve_neg().contiguous() : g.contiguous());
        list.push_back({held.back().data_ptr(), g.numel(), dtype_of(g), 0});
    }
    const Tensor norm = at::empty({}, first.options().dtype(at::kFloat)), work = work_of(ok(mo_gradient_work((int64_t)list.size()), "mo_gradient_work"), first);
    ok(mo_gradient_norm(list.data(), (int64_t)list.size(), scale, (float)max_norm, (float)eps, data(norm), data<void>(work), stream_of(first)), "mo_gradient_norm");
    if (scale)
        for (size_t i = 0; i < given.size(); i++) {
            if (list[i].p == given[i].data_ptr()) written(given[i]);
            else given[i].copy_(held[i]);
        }
    return norm;
}

}  // namespace

PYBIND11_MODULE(_mario_ops_torch, m) {
    m.def("attend", &attend, py::call_guard<py::gil_scoped_release>());
    m.def("attend_step", &attend_step, py::call_guard<py::gil_scoped_release>());
    m.def("group_norm_act", &group_norm_act, py::call_guard<py::gil_scoped_release>());
    m.def("conv", &conv, py::call_guard<py::gil_scoped_release>());
    m.def("conv_step", &conv_step, py::call_guard<py::gil_scoped_release>());
    m.def("scan", &scan, py::call_guard<py::gil_scoped_release>());
    m.def("scan_step", &scan_step, py::call_guard<py::gil_scoped_release>());
    m.def("gradient_norm", &gradient_norm, py::call_guard<py::gil_scoped_release>());
}
