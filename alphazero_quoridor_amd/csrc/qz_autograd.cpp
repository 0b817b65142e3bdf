// qz_autograd.cpp -- the autograd side of the policy losses (losses.py), host code only.  Written in C++ because a Python
// autograd function costs more than the kernels at the sizes of a training minibatch: its backward pass has to win the
// interpreter's lock on the engine's thread (105 us for 128 x 140 with a gradient, 197 us before the call's host work was cut).
// Arguments are checked in losses.py; every tensor here is two- or one-dimensional with contiguous rows.
#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>
#include <c10/core/DeviceGuard.h>
#include <torch/extension.h>

#include "../../include/qz_abi.h"

namespace {

using torch::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

void* stream_of(const Tensor& t) { return c10::hip::getCurrentHIPStreamMasqueradingAsCUDA(t.device().index()).stream(); }
void check(int rc) { TORCH_CHECK(rc == 0, "libqzero_hip error ", rc, ": ", qz_last_error()); }
// a backward pass under create_graph would return a gradient that autograd takes for a constant
void refuse_twice() { TORCH_CHECK(!at::GradMode::is_enabled(), "the policy losses can be differentiated once only (create_graph is not supported)"); }
// A dual tensor requires no gradient, so the functions below would compute on its values and drop its tangent without a word.
void refuse_tangents(std::initializer_list<Tensor> inputs) {
    if (!c10::AutogradState::get_tls_state().get_fw_grad_mode()) return;
    for (const Tensor& t : inputs)
        TORCH_CHECK_NOT_IMPLEMENTED(!t.defined() || !t._fw_grad(/*level=*/0).defined(), "the policy losses have no forward-mode derivative");
}
// (a lazily negated view's memory holds the values of the other sign)
Tensor plain(const Tensor& t) { return t.resolve_neg().contiguous(); }
void* ptr(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
float* fptr(const Tensor& t) { return static_cast<float*>(ptr(t)); }
int dtype_of(const Tensor& t) { return t.scalar_type() == at::kFloat ? QZ_F32 : t.scalar_type() == at::kBFloat16 ? QZ_BF16 : QZ_F16; }

qz_policy_rows rows_of(const Tensor& z, const Tensor& actions, const Tensor& legal, int64_t kind) {
    qz_policy_rows r;
    r.logits = z.data_ptr();
    r.ld = z.stride(0);
    r.n = z.size(0);
    r.n_actions = (int32_t)z.size(1);
    r.dtype = dtype_of(z);
    r.actions = static_cast<const int64_t*>(actions.data_ptr());
    r.legal = ptr(legal);
    r.legal_ld = legal.defined() ? legal.stride(0) : 0;
    r.legal_kind = (int32_t)kind;
    return r;
}
struct LossArgs {
    Tensor actions, legal, adv, old_logp, ref_logp, weights, ref;  // legal and the last three may be undefined
    int64_t kind;
    double lo, hi, kl, ent;
};
qz_policy_terms terms_of(const LossArgs& a) {
    qz_policy_terms t;
    t.advantages = fptr(a.adv);
    t.old_logp = fptr(a.old_logp);
    t.ref_logp = fptr(a.ref_logp);
    t.weights = fptr(a.weights);
    t.ref_logits = ptr(a.ref);
    t.ref_ld = a.ref.defined() ? a.ref.stride(0) : 0;
    t.clip_low = (float)a.lo;
    t.clip_high = (float)a.hi;
    t.kl_coef = (float)a.kl;
    t.entropy_coef = (float)a.ent;
    return t;
}
// The graph capture that the current stream records into; 0: none, -1: it cannot be told.
int64_t capture_of(const Tensor& z) {
    hipStreamCaptureStatus status = hipStreamCaptureStatusNone;
    unsigned long long id = 0;
    if (hipStreamGetCaptureInfo(static_cast<hipStream_t>(stream_of(z)), &status, &id) != hipSuccess) {
        (void)hipGetLastError();
        return -1;
    }
    return status == hipStreamCaptureStatusNone ? 0 : (int64_t)id;
}
Tensor scratch(const Tensor& z, int64_t bytes) { return at::empty({bytes > 0 ? bytes : 1}, z.options().dtype(at::kByte)); }

// ---- log-probabilities.  -> logp, entropy (undefined unless asked for), statistics (undefined unless asked for)
std::tuple<Tensor, Tensor, Tensor> run_logp(const Tensor& z, const Tensor& actions, const Tensor& legal, int64_t kind, bool entropy, bool stats) {
    const c10::DeviceGuard guard(z.device());
    const auto f32 = z.options().dtype(at::kFloat);
    const int64_t n = z.size(0), bytes = qz_policy_workspace(n, (int)z.size(1));
    Tensor logp = at::empty({n}, f32), h, st, ws = scratch(z, bytes);
    if (entropy) h = at::empty({n}, f32);
    if (stats) st = at::empty({2, n}, f32);
    const qz_policy_rows r = rows_of(z, actions, legal, kind);
    check(qz_action_logp(&r, fptr(logp), fptr(h), fptr(st), ws.data_ptr(), bytes, stream_of(z)));
    return {logp, h, st};
}
// (what is constant to autograd travels in a struct: an autograd function's tensor arguments may not be undefined)
struct LogpArgs {
    Tensor actions, legal;
    int64_t kind;
    bool entropy;
};
struct ActionLogp : torch::autograd::Function<ActionLogp> {
    static variable_list forward(AutogradContext* ctx, const Tensor& z, const LogpArgs& a) {
        auto [logp, h, st] = run_logp(z, a.actions, a.legal, a.kind, a.entropy, true);
        ctx->save_for_backward({z, a.actions, a.legal, st, h});
        ctx->saved_data["kind"] = a.kind;
        ctx->set_materialize_grads(false);
        return a.entropy ? variable_list{logp, h} : variable_list{logp};
    }
    static variable_list backward(AutogradContext* ctx, variable_list up) {
        refuse_twice();
        const auto saved = ctx->get_saved_variables();
        const Tensor &z = saved[0], &h = saved[4];
        const Tensor dlogp = up[0].defined() ? plain(up[0]) : Tensor(), dh = up.size() > 1 && up[1].defined() ? plain(up[1]) : Tensor();
        Tensor grad;
        if (dlogp.defined() || dh.defined()) {
            const c10::DeviceGuard guard(z.device());
            grad = at::empty({z.size(0), z.size(1)}, z.options());
            const qz_policy_rows r = rows_of(z, saved[1], saved[2], ctx->saved_data["kind"].toInt());
            check(qz_action_logp_backward(&r, fptr(saved[3]), fptr(h), fptr(dlogp), fptr(dh), grad.data_ptr(), grad.size(1), stream_of(z)));
        }
        return {grad, Tensor()};
    }
};
std::tuple<Tensor, Tensor> action_logp(const Tensor& z, const Tensor& actions, const std::optional<Tensor>& legal, int64_t kind, bool entropy) {
    const Tensor mask = legal.value_or(Tensor());
    refuse_tangents({z});
    if (at::GradMode::is_enabled() && z.requires_grad()) {
        const variable_list out = ActionLogp::apply(z, LogpArgs{actions, mask, kind, entropy});
        return {out[0], entropy ? out[1] : Tensor()};
    }
    auto [logp, h, st] = run_logp(z, actions, mask, kind, entropy, false);
    return {logp, h};
}

// ---- the clipped loss.  -> loss, logp, kl, entropy, gradient (undefined unless asked for), workspace
struct LossOut {
    Tensor loss, logp, kl, entropy, grad, ws;
};
LossOut run_loss(const Tensor& z, const LossArgs& a, bool want_grad) {
    const c10::DeviceGuard guard(z.device());
    const qz_policy_rows r = rows_of(z, a.actions, a.legal, a.kind);
    const qz_policy_terms t = terms_of(a);
    const auto f32 = z.options().dtype(at::kFloat);
    const int64_t n = r.n, bytes = qz_policy_workspace(n, r.n_actions);
    LossOut o;
    Tensor rows = at::empty({3, n}, f32);
    o.loss = at::empty({}, f32);
    o.logp = rows.select(0, 0);
    o.kl = rows.select(0, 1);
    o.entropy = rows.select(0, 2);
    o.ws = scratch(z, bytes);
    if (want_grad) o.grad = at::empty({n, z.size(1)}, z.options());
    float* at_ = fptr(rows);
    check(qz_policy_loss(&r, &t, fptr(o.loss), at_, at_ + n, at_ + 2 * n, ptr(o.grad), z.size(1), o.ws.data_ptr(), bytes, stream_of(z)));
    return o;
}
// The forward pass writes the gradient for an upstream factor of 1 beside the loss (one pass over the logits for both); the backward
// pass hands it out, or computes it again where the factor is another, it was handed out before, or the backward pass is recorded into
// a graph that does not hold the forward pass: its replays would all find what the forward pass wrote once.
struct PolicyLoss : torch::autograd::Function<PolicyLoss> {
    static variable_list forward(AutogradContext* ctx, const Tensor& z, const LossArgs& a) {
        LossOut o = run_loss(z, a, true);
        ctx->save_for_backward({z, a.actions, a.legal, a.adv, a.old_logp, a.ref_logp, a.weights, a.ref});
        ctx->saved_data["kind"] = a.kind;
        ctx->saved_data["coef"] = std::vector<double>{a.lo, a.hi, a.kl, a.ent};
        ctx->saved_data["grad"] = o.grad;
        ctx->saved_data["ws"] = o.ws;
        ctx->saved_data["capture"] = capture_of(z);
        ctx->mark_non_differentiable({o.logp, o.kl, o.entropy});
        ctx->set_materialize_grads(false);
        return {o.loss, o.logp, o.kl, o.entropy};
    }
    static variable_list backward(AutogradContext* ctx, variable_list up) {
        refuse_twice();
        const auto s = ctx->get_saved_variables();  // (checks that none of them was changed in place)
        variable_list out(2);
        if (!up[0].defined()) return out;
        const Tensor& z = s[0];
        const c10::DeviceGuard guard(z.device());
        const auto c = ctx->saved_data["coef"].toDoubleVector();
        Tensor grad = ctx->saved_data["grad"].toTensor(), ws = ctx->saved_data["ws"].toTensor();
        ctx->saved_data["grad"] = Tensor();
        const int64_t capture = capture_of(z);
        const bool kept = grad.defined() && capture >= 0 && capture == ctx->saved_data["capture"].toInt();
        const int64_t bytes = qz_policy_workspace(z.size(0), (int)z.size(1));
        if (!kept) {  // computed again, with a workspace of its own
            grad = at::empty({z.size(0), z.size(1)}, z.options());
            ws = scratch(z, bytes);
        }
        const Tensor upstream = plain(up[0]);
        const LossArgs a = {s[1], s[2], s[3], s[4], s[5], s[6], s[7], ctx->saved_data["kind"].toInt(), c[0], c[1], c[2], c[3]};
        const qz_policy_rows r = rows_of(z, a.actions, a.legal, a.kind);
        const qz_policy_terms t = terms_of(a);
        check(qz_policy_loss_backward(&r, &t, fptr(upstream), kept, grad.data_ptr(), grad.size(1), ws.data_ptr(), bytes, stream_of(z)));
        out[0] = grad;
        return out;
    }
};
using Maybe = std::optional<Tensor>;
std::tuple<Tensor, Tensor, Tensor, Tensor, Maybe> policy_loss(const Tensor& z, const Tensor& actions, const Maybe& legal, int64_t kind, const Tensor& adv,
                                                              const Tensor& old_logp, const Maybe& ref_logp, const Maybe& weights, const Maybe& ref, double lo,
                                                              double hi, double kl, double ent, bool raw_grad) {
    const LossArgs a = {actions, legal.value_or(Tensor()), adv, old_logp, ref_logp.value_or(Tensor()), weights.value_or(Tensor()), ref.value_or(Tensor()), kind, lo, hi, kl, ent};
    refuse_tangents({z, adv, old_logp, a.ref_logp, a.weights, a.ref});
    if (!raw_grad && at::GradMode::is_enabled() && z.requires_grad()) {
        const variable_list o = PolicyLoss::apply(z, a);
        return {o[0], o[1], o[2], o[3], Maybe()};
    }
    LossOut o = run_loss(z, a, raw_grad);
    return {o.loss, o.logp, o.kl, o.entropy, raw_grad ? Maybe(o.grad) : Maybe()};
}

}  // namespace

PYBIND11_MODULE(_autograd, m) {
    m.doc() = "autograd functions over the policy-loss entry points of libqzero_hip.so; see losses.py";
    // (the interpreter's lock is given up: the calls allocate and launch, and touch no Python object)
    m.def("action_logp", &action_logp, py::call_guard<py::gil_scoped_release>());
    m.def("policy_loss", &policy_loss, py::call_guard<py::gil_scoped_release>());
}
