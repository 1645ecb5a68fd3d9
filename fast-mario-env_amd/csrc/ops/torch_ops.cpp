// The operators of libmario_ops.so on torch tensors: allocation, views, streams and autograd. Their host work is most of a small
// call's time, and in a training step it runs on autograd's own thread, so none of it is left to Python. Arguments come checked
// (memory.py): plain tensors of one GPU with the types and shapes that include/mario_ops.h asks for.
#include <ATen/ATen.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/utils/pybind.h>

#include <optional>

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
    if (!state.is_inference()) state.unsafeGetTensorImpl()->bump_version();   // (what saved it for a gradient notices)
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

}  // namespace

PYBIND11_MODULE(_mario_ops_torch, m) {
    m.def("attend", &attend, py::call_guard<py::gil_scoped_release>());
    m.def("attend_step", &attend_step, py::call_guard<py::gil_scoped_release>());
    m.def("group_norm_act", &group_norm_act, py::call_guard<py::gil_scoped_release>());
}
