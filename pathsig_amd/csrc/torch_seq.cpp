// Registration of the sequence operators (linear attention with decays, norms before and after a block) with the torch
// dispatcher: schemas, argument checks, device implementations over the C ABI of pathsig_hip.h, autograd nodes, and the
// functions that plain eager calls take past the dispatcher.  They have no counterpart in the reference.
#include <algorithm>
#include <array>
#include <optional>
#include <tuple>
#include <vector>

#include <torch/csrc/autograd/autograd_not_implemented_fallback.h>

#include "torch_common.hpp"

namespace psig_torch {
namespace {

using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
using MaybeTensor = std::optional<Tensor>;

Tensor or_undefined(const MaybeTensor &t) { return t.has_value() ? *t : Tensor(); }
// (an operator returns tensors: an empty one for what was not asked for)
Tensor or_empty(const Tensor &t, const Tensor &like) { return t.defined() ? t : at::empty({0}, like.options()); }
MaybeTensor or_none(const Tensor &t) { return t.defined() ? MaybeTensor(t) : MaybeTensor(); }

int sequence_dtype(const Tensor &t, const char *what) {
    if (t.scalar_type() == at::kFloat) return PATHSIG_F32;
    if (t.scalar_type() == at::kBFloat16) return PATHSIG_BF16;
    TORCH_CHECK(false, what, " must be float32 or bfloat16");
}

void check_like(const Tensor &t, const char *what, const Tensor &like, const char *like_name) {
    TORCH_CHECK(t.is_cuda(), what, " must be CUDA");
    TORCH_CHECK(t.device() == like.device(), what, " must be on the device of ", like_name);
}

// The channels of a head side by side, tokens no further apart than the kernels' offsets reach, and a start at a multiple of 16
// bytes (of sequences, whose rows are read in such units).
Tensor side_by_side(const Tensor &t, bool sequence) {
    const bool near = !sequence || t.size(1) <= 1 || t.stride(1) <= PATHSIG_MAX_TOKEN_STRIDE;
    const Tensor as = near && (t.size(-1) == 1 || t.stride(-1) == 1) ? t : t.contiguous();
    return sequence && (uintptr_t)ptr(as) % 16 ? as.clone(at::MemoryFormat::Contiguous) : as;
}

// ---- linear attention ---------------------------------------------------------------------------------------------
struct AttentionCall {
    Tensor q, k, v, log_decay, state, lengths;
    pathsig_linattn c;
};

// (the stride of an axis of one is anything, and never used)
int64_t stride_of(const Tensor &t, int64_t axis) { return t.size(axis) > 1 ? t.stride(axis) : 0; }

void set_strides(int64_t (&out)[3], const Tensor &t, bool token) {
    out[0] = stride_of(t, 0);
    out[1] = token ? stride_of(t, 1) : 0;
    out[2] = stride_of(t, token ? 2 : 1);
}

// token: q is [B, L, H, D] and so on; else [B, H, D], one token of every sequence
AttentionCall attention_call(const Tensor &q, const Tensor &k, const Tensor &v, const Tensor &log_decay, const Tensor &state,
                             const Tensor &lengths, double scale, bool token) {
    AttentionCall a;
    const int64_t dims = token ? 4 : 3;
    const char *const shape = token ? "[B, L, heads, D]" : "[B, heads, D]";
    TORCH_CHECK(q.is_cuda(), "q must be CUDA");
    a.c = {};
    a.c.dtype = sequence_dtype(q, "q");
    TORCH_CHECK(q.dim() == dims, "q must be ", shape);
    for (const auto &[t, name] : {std::pair<const Tensor *, const char *>{&k, "k"}, {&v, "v"}}) {
        check_like(*t, name, q, "q");
        TORCH_CHECK(t->scalar_type() == q.scalar_type(), name, " must have same dtype as q");
        TORCH_CHECK(t->dim() == dims, name, " must be ", shape);
        for (int64_t i = 0; i < dims - 2; ++i)
            TORCH_CHECK(t->size(i) == q.size(i), name, " must have as many sequences and tokens as q");
    }
    const int64_t heads = dims - 2;
    TORCH_CHECK(k.size(heads) == v.size(heads), "k and v must have the same number of heads");
    TORCH_CHECK(k.size(dims - 1) == q.size(dims - 1), "k must have as many channels as q");
    a.c.B = q.size(0);
    a.c.L = token ? q.size(1) : 1;
    a.c.H = q.size(heads);
    a.c.Hkv = k.size(heads);
    a.c.Dk = q.size(dims - 1);
    a.c.Dv = v.size(dims - 1);
    TORCH_CHECK(a.c.H >= 1 && a.c.Hkv >= 1 && a.c.H % a.c.Hkv == 0, "the heads of q must be a multiple of those of k and v");
    check_like(log_decay, "log_decay", q, "q");
    TORCH_CHECK(log_decay.scalar_type() == at::kFloat, "log_decay must be float32");
    TORCH_CHECK(log_decay.dim() == 1 && log_decay.size(0) == a.c.H, "log_decay must be [heads of q]");
    a.q = side_by_side(q, token);
    a.k = side_by_side(k, token);
    a.v = side_by_side(v, token);
    a.log_decay = log_decay.contiguous();
    if (state.defined()) {
        check_like(state, "state", q, "q");
        TORCH_CHECK(state.scalar_type() == at::kFloat, "state must be float32");
        TORCH_CHECK(state.sizes() == at::IntArrayRef({a.c.B, a.c.H, a.c.Dk, a.c.Dv}), "state must be [B, heads of q, Dk, Dv]");
        a.state = state.contiguous();
    }
    if (lengths.defined()) {
        check_like(lengths, "lengths", q, "q");
        TORCH_CHECK(lengths.scalar_type() == at::kInt || lengths.scalar_type() == at::kLong, "lengths must be int32 or int64");
        TORCH_CHECK(lengths.dim() == 1 && lengths.size(0) == a.c.B, "lengths must be [B]");
        // (clamped before it is narrowed: a length is anything up to the largest int64)
        a.lengths = (lengths.scalar_type() == at::kInt ? lengths : lengths.clamp(0, a.c.L).to(at::kInt)).contiguous();
    }
    set_strides(a.c.q_stride, a.q, token);
    set_strides(a.c.k_stride, a.k, token);
    set_strides(a.c.v_stride, a.v, token);
    a.c.scale = (float)scale;
    a.c.log_decay = (const float *)ptr(a.log_decay);
    a.c.lengths = (const int32_t *)ptr(a.lengths);
    return a;
}

// (out, last state or undefined, the workspace: what the backward of the same call can use again, or undefined)
std::tuple<Tensor, Tensor, Tensor> attention_forward(const Tensor &q, const Tensor &k, const Tensor &v, const Tensor &log_decay,
                                                     const Tensor &state, const Tensor &lengths, double scale, bool return_state,
                                                     bool learned_decay) {
    c10::DeviceGuard guard(q.device());
    AttentionCall a = attention_call(q, k, v, log_decay, state, lengths, scale, true);
    a.c.learned_decay = learned_decay;
    Tensor out = at::empty({a.c.B, a.c.L, a.c.H, a.c.Dv}, a.q.options());
    Tensor last = return_state ? at::empty({a.c.B, a.c.H, a.c.Dk, a.c.Dv}, a.log_decay.options()) : Tensor();
    const size_t ws_bytes = pathsig_linattn_forward_workspace(&a.c);
    Tensor ws = scratch(ws_bytes, a.q);
    check_rc(pathsig_linattn_forward(&a.c, ptr(a.q), ptr(a.k), ptr(a.v), (const float *)ptr(a.state), ptr(out),
                                     (float *)ptr(last), ptr(ws), ws_bytes, stream_of(a.q)));
    return {out, last, ws};
}

using Gradients = std::tuple<Tensor, Tensor, Tensor, Tensor, Tensor>;

// which gradients are asked for; empty tensors stand for the others
struct Wanted {
    bool q = true, k = true, v = true, decay = false, state = false;
};

Gradients attention_backward(const Tensor &grad_out_in, const Tensor &grad_last_in, const Tensor &q, const Tensor &k,
                             const Tensor &v, const Tensor &log_decay, const Tensor &state, const Tensor &lengths,
                             const Tensor &kept, double scale, const Wanted &want) {
    c10::DeviceGuard guard(q.device());
    AttentionCall a = attention_call(q, k, v, log_decay, state, lengths, scale, true);
    a.c.learned_decay = want.decay;
    check_like(grad_out_in, "grad_out", q, "q");
    TORCH_CHECK(grad_out_in.scalar_type() == q.scalar_type(), "grad_out must have same dtype as q");
    TORCH_CHECK(grad_out_in.sizes() == at::IntArrayRef({a.c.B, a.c.L, a.c.H, a.c.Dv}), "grad_out must be [B, L, H, Dv]");
    Tensor grad_out = side_by_side(grad_out_in.contiguous(), true), grad_last;
    if (grad_last_in.defined()) {
        check_like(grad_last_in, "grad_state", q, "q");
        TORCH_CHECK(grad_last_in.scalar_type() == at::kFloat, "grad_state must be float32");
        TORCH_CHECK(grad_last_in.sizes() == at::IntArrayRef({a.c.B, a.c.H, a.c.Dk, a.c.Dv}), "grad_state must be [B, H, Dk, Dv]");
        grad_last = grad_last_in.contiguous();
    }
    auto gradient = [](bool wanted, at::IntArrayRef shape, const Tensor &like) {
        return at::empty(wanted ? shape : at::IntArrayRef({0}), like.options());
    };
    const Tensor dq = gradient(want.q, {a.c.B, a.c.L, a.c.H, a.c.Dk}, a.q), dk = gradient(want.k, {a.c.B, a.c.L, a.c.Hkv, a.c.Dk}, a.q),
                 // (from the sweep of the state's gradient)
                 dv = gradient(want.v || want.state, {a.c.B, a.c.L, a.c.Hkv, a.c.Dv}, a.q),
                 ddecay = gradient(want.decay, {a.c.H}, a.log_decay),
                 dstate = gradient(want.state, {a.c.B, a.c.H, a.c.Dk, a.c.Dv}, a.log_decay);
    const size_t ws_bytes = pathsig_linattn_backward_workspace(&a.c, want.decay);
    Tensor ws = scratch(ws_bytes, a.q);
    // The forward's workspace holds copies of q, k and v where they did not lie in whole units.  Hooks on saved tensors may hand them
    // back in other strides: a workspace that is not this call's is left, and worked out again.
    const size_t kept_bytes = pathsig_linattn_forward_workspace(&a.c);
    const bool use = kept.defined() && kept.is_contiguous() && (size_t)kept.nbytes() == kept_bytes && kept.device() == q.device() &&
                     (uintptr_t)ptr(kept) % 16 == 0;
    check_rc(pathsig_linattn_backward(&a.c, ptr(a.q), ptr(a.k), ptr(a.v), (const float *)ptr(a.state), use ? ptr(kept) : nullptr,
                                      use ? kept_bytes : 0, ptr(grad_out), (const float *)ptr(grad_last), ptr(dq), ptr(dk), ptr(dv),
                                      (float *)ptr(ddecay), (float *)ptr(dstate), ptr(ws), ws_bytes, stream_of(a.q)));
    return {dq, dk, dv, ddecay, dstate};
}

Tensor attention_step(const Tensor &q, const Tensor &k, const Tensor &v, const Tensor &log_decay, const Tensor &state,
                      double scale) {
    c10::DeviceGuard guard(q.device());
    TORCH_CHECK(state.defined() && state.is_contiguous(), "state is updated in place: it must be contiguous");
    const AttentionCall a = attention_call(q, k, v, log_decay, state, Tensor(), scale, false);
    Tensor out = at::empty({a.c.B, a.c.H, a.c.Dv}, a.q.options());
    torch::autograd::impl::bump_version(state);  // (first: it refuses an inference tensor outside of inference mode)
    check_rc(pathsig_linattn_step(&a.c, ptr(a.q), ptr(a.k), ptr(a.v), (float *)ptr(a.state), ptr(out), stream_of(a.q)));
    return out;
}

std::tuple<Tensor, Tensor> linear_attention_hip(const Tensor &q, const Tensor &k, const Tensor &v, const Tensor &log_decay,
                                                const MaybeTensor &state, const MaybeTensor &lengths, double scale,
                                                bool return_state) {
    auto [out, last, kept] =
        attention_forward(q, k, v, log_decay, or_undefined(state), or_undefined(lengths), scale, return_state, false);
    return {out, or_empty(last, log_decay)};
}

Gradients linear_attention_backward_hip(const Tensor &grad_out, const MaybeTensor &grad_state, const Tensor &q, const Tensor &k,
                                        const Tensor &v, const Tensor &log_decay, const MaybeTensor &state,
                                        const MaybeTensor &lengths, double scale, bool want_log_decay, bool want_state) {
    return attention_backward(grad_out, or_undefined(grad_state), q, k, v, log_decay, or_undefined(state), or_undefined(lengths),
                              Tensor(), scale, {true, true, true, want_log_decay, want_state});
}

bool any_grad(std::initializer_list<const Tensor *> all) {
    if (!at::GradMode::is_enabled()) return false;
    for (const Tensor *t : all)
        if (t->defined() && t->requires_grad()) return true;
    return false;
}

Tensor linear_attention_step_hip(const Tensor &q, const Tensor &k, const Tensor &v, const Tensor &log_decay, Tensor state,
                                 double scale) {
    return attention_step(q, k, v, log_decay, state, scale);
}

using AttentionOp = std::tuple<Tensor, Tensor>(const Tensor &, const Tensor &, const Tensor &, const Tensor &,
                                               const MaybeTensor &, const MaybeTensor &, double, bool);
using AttentionBackwardOp = Gradients(const Tensor &, const MaybeTensor &, const Tensor &, const Tensor &, const Tensor &,
                                      const Tensor &, const MaybeTensor &, const MaybeTensor &, double, bool, bool);
using StepOp = Tensor(const Tensor &, const Tensor &, const Tensor &, const Tensor &, Tensor, double);

// DIRECT: the device implementations are called past the dispatcher (plain tensors in plain eager mode); a backward that meets
// anything else, or is asked for a graph of the gradient, takes the operator
template <bool DIRECT>
struct AttentionFunction : public torch::autograd::Function<AttentionFunction<DIRECT>> {
    static variable_list forward(AutogradContext *ctx, const Tensor &q, const Tensor &k, const Tensor &v, const Tensor &log_decay,
                                 const MaybeTensor &maybe_state, const MaybeTensor &maybe_lengths, double scale,
                                 bool return_state) {
        at::AutoDispatchBelowADInplaceOrView below;
        const Tensor state = or_undefined(maybe_state), lengths = or_undefined(maybe_lengths);
        Tensor out, last, kept;
        if constexpr (DIRECT) {
            std::tie(out, last, kept) =
                attention_forward(q, k, v, log_decay, state, lengths, scale, return_state, log_decay.requires_grad());
        } else {
            static auto op = typed_op<AttentionOp>("pathsig::linear_attention");
            std::tie(out, last) = op.call(q, k, v, log_decay, maybe_state, maybe_lengths, scale, return_state);
        }
        ctx->save_for_backward({q, k, v, log_decay, state, lengths, kept});
        ctx->saved_data["scale"] = scale;
        ctx->set_materialize_grads(false);
        if (DIRECT && !return_state) return {out};
        if (!return_state) ctx->mark_non_differentiable({last});
        return {out, last};
    }
    static variable_list backward(AutogradContext *ctx, variable_list grads) {
        variable_list out(8);
        const Tensor grad_last = grads.size() > 1 ? grads[1] : Tensor();
        if (!grads[0].defined() && !grad_last.defined()) return out;
        const auto saved = ctx->get_saved_variables();
        const Tensor &q = saved[0], &k = saved[1], &v = saved[2], &log_decay = saved[3], &state = saved[4], &lengths = saved[5],
                     &kept = saved[6];
        const double scale = ctx->saved_data["scale"].toDouble();
        Tensor grad_out = grads[0];
        if (!grad_out.defined()) grad_out = at::zeros({q.size(0), q.size(1), q.size(2), v.size(3)}, q.options());
        const Wanted want{ctx->needs_input_grad(0), ctx->needs_input_grad(1), ctx->needs_input_grad(2), ctx->needs_input_grad(3),
                          state.defined() && ctx->needs_input_grad(4)};
        bool direct = DIRECT && !at::GradMode::is_enabled();
        for (const Tensor *t : {(const Tensor *)&grad_out, &q, &k, &v, &log_decay}) direct = direct && plain(*t);
        for (const Tensor *t : {&state, &lengths, &kept, &grad_last}) direct = direct && (!t->defined() || plain(*t));
        Gradients g;
        if (direct) {
            g = attention_backward(grad_out, grad_last, q, k, v, log_decay, state, lengths, kept, scale, want);
        } else {
            static auto op = typed_op<AttentionBackwardOp>("pathsig::linear_attention_backward");
            g = op.call(grad_out, or_none(grad_last), q, k, v, log_decay, or_none(state), or_none(lengths), scale, want.decay,
                        want.state);
        }
        if (want.q) out[0] = std::get<0>(g);
        if (want.k) out[1] = std::get<1>(g);
        if (want.v) out[2] = std::get<2>(g);
        if (want.decay) out[3] = std::get<3>(g);
        if (want.state) out[4] = std::get<4>(g);
        return out;
    }
};

std::tuple<Tensor, Tensor> linear_attention_autograd(const Tensor &q, const Tensor &k, const Tensor &v, const Tensor &log_decay,
                                                     const MaybeTensor &state, const MaybeTensor &lengths, double scale,
                                                     bool return_state) {
    auto out = AttentionFunction<false>::apply(q, k, v, log_decay, state, lengths, scale, return_state);
    return {out[0], out[1]};
}

Tensor linear_attention_step_autograd(const Tensor &q, const Tensor &k, const Tensor &v, const Tensor &log_decay, Tensor state,
                                      double scale) {
    TORCH_CHECK(!any_grad({&q, &k, &v, &log_decay, &state}),
                "linear_attention_step has no gradient: call it under torch.no_grad(), or linear_attention for training");
    at::AutoDispatchBelowADInplaceOrView below;
    static auto op = typed_op<StepOp>("pathsig::linear_attention_step");
    return op.call(q, k, v, log_decay, state, scale);
}

// ---- norms --------------------------------------------------------------------------------------------------------
struct NormCall {
    Tensor x, gate, residual, weight, scale, next_weight;
    pathsig_norm c;
    std::vector<int64_t> shape;
};

// rows of C channels side by side at one distance from each other, without a copy where the tensor allows it
Tensor as_rows(const Tensor &t, int64_t C) {
    const Tensor rows = t.reshape({t.numel() / C, C});
    return C == 1 || rows.stride(1) == 1 ? rows : rows.contiguous();
}

NormCall norm_call(const Tensor &x, const Tensor &weight, const Tensor &gate, const Tensor &residual, const Tensor &scale,
                   const Tensor &next_weight, double eps, int64_t activation) {
    NormCall a;
    a.c = {};
    TORCH_CHECK(x.is_cuda(), "x must be CUDA");
    a.c.dtype = sequence_dtype(x, "x");
    a.c.param_dtype = a.c.dtype;
    TORCH_CHECK(x.dim() >= 1 && x.size(-1) >= 1, "x must be [..., C] with at least one channel");
    const int64_t C = x.size(-1);
    a.shape = x.sizes().vec();
    a.x = as_rows(x, C);
    for (const auto &[t, name, to] : {std::tuple<const Tensor *, const char *, Tensor *>{&gate, "gate", &a.gate},
                                      {&residual, "residual", &a.residual}}) {
        if (!t->defined()) continue;
        check_like(*t, name, x, "x");
        TORCH_CHECK(t->scalar_type() == x.scalar_type(), name, " must have same dtype as x");
        TORCH_CHECK(t->sizes() == x.sizes(), name, " must have the shape of x");
        *to = as_rows(*t, C);
    }
    bool first = true;
    for (const auto &[t, name, to] : {std::tuple<const Tensor *, const char *, Tensor *>{&weight, "weight", &a.weight},
                                      {&scale, "scale", &a.scale},
                                      {&next_weight, "next_weight", &a.next_weight}}) {
        if (!t->defined()) continue;
        check_like(*t, name, x, "x");
        TORCH_CHECK(t->dim() == 1 && t->size(0) == C, name, " must be [C]");
        TORCH_CHECK(t->scalar_type() == at::kFloat || t->scalar_type() == x.scalar_type(), name,
                    " must be float32 or have the dtype of x");
        const int code = t->scalar_type() == at::kFloat ? PATHSIG_F32 : a.c.dtype;
        TORCH_CHECK(first || code == a.c.param_dtype, "weight, scale and next_weight must have one dtype");
        a.c.param_dtype = code;
        first = false;
        *to = t->contiguous();
    }
    TORCH_CHECK(activation >= PATHSIG_GATE_SILU && activation <= PATHSIG_GATE_LINEAR, "unknown activation");
    a.c.activation = (int)activation;
    a.c.rows = a.x.size(0);
    a.c.C = C;
    a.c.x_stride = a.x.stride(0);
    a.c.gate_stride = a.gate.defined() ? a.gate.stride(0) : 0;
    a.c.residual_stride = a.residual.defined() ? a.residual.stride(0) : 0;
    a.c.eps = (float)eps;
    a.c.x = ptr(a.x);
    a.c.gate = ptr(a.gate);
    a.c.residual = ptr(a.residual);
    a.c.weight = ptr(a.weight);
    a.c.scale = ptr(a.scale);
    a.c.next_weight = ptr(a.next_weight);
    return a;
}

// (out, next, statistics): next and statistics are undefined where they are not wanted
std::tuple<Tensor, Tensor, Tensor> norm_forward(const Tensor &x, const Tensor &weight, const Tensor &gate, const Tensor &residual,
                                                const Tensor &scale, const Tensor &next_weight, double eps, int64_t activation,
                                                bool keep) {
    c10::DeviceGuard guard(x.device());
    const NormCall a = norm_call(x, weight, gate, residual, scale, next_weight, eps, activation);
    Tensor out = at::empty(a.shape, x.options());
    Tensor next = next_weight.defined() ? at::empty(a.shape, x.options()) : Tensor();
    Tensor stats = keep ? at::empty({2, a.c.rows}, x.options().dtype(at::kFloat)) : Tensor();
    check_rc(pathsig_norm_forward(&a.c, ptr(out), ptr(next), (float *)ptr(stats), stream_of(x)));
    return {out, next, stats};
}

using NormGradients = std::tuple<Tensor, Tensor, Tensor, Tensor, Tensor, Tensor>;

// gradients of x, weight, gate, residual, scale, next_weight, those that are wanted; an empty tensor for what is not, or is not there
NormGradients norm_backward(const Tensor &grad_out, const Tensor &grad_next, const Tensor &x, const Tensor &weight,
                            const Tensor &gate, const Tensor &residual, const Tensor &scale, const Tensor &next_weight,
                            const Tensor &stats, double eps, int64_t activation, const std::array<bool, 6> &want) {
    c10::DeviceGuard guard(x.device());
    const NormCall a = norm_call(x, weight, gate, residual, scale, next_weight, eps, activation);
    Tensor up[2];
    for (int i = 0; i < 2; ++i) {
        const Tensor &g = i == 0 ? grad_out : grad_next;
        if (!g.defined()) continue;
        check_like(g, "the gradient from above", x, "x");
        TORCH_CHECK(g.scalar_type() == x.scalar_type() && g.sizes() == x.sizes(),
                    "the gradient from above must have the dtype and shape of x");
        up[i] = g.contiguous();
    }
    check_like(stats, "statistics", x, "x");
    TORCH_CHECK(stats.scalar_type() == at::kFloat && stats.is_contiguous() && stats.dim() == 2 && stats.size(0) == 2 &&
                    stats.size(1) == a.c.rows,
                "statistics must be the forward's");
    const at::TensorOptions params = x.options().dtype(a.c.param_dtype == PATHSIG_F32 ? at::kFloat : x.scalar_type());
    auto rows = [&](const Tensor &t, bool wanted) {
        return at::empty(wanted && t.defined() ? at::IntArrayRef(a.shape) : at::IntArrayRef({0}), x.options());
    };
    auto column = [&](const Tensor &t, bool wanted) { return at::empty({wanted && t.defined() ? a.c.C : 0}, params); };
    const Tensor dx = rows(x, want[0]), dweight = column(weight, want[1]), dgate = rows(gate, want[2]), dresidual = rows(residual, want[3]),
                 dscale = column(scale, want[4]), dnext = column(next_weight, want[5]);
    const size_t ws_bytes = pathsig_norm_backward_workspace(&a.c);
    Tensor ws = dweight.numel() + dscale.numel() + dnext.numel() > 0 ? scratch(ws_bytes, x) : Tensor();
    check_rc(pathsig_norm_backward(&a.c, (const float *)ptr(stats), ptr(up[0]), ptr(up[1]), ptr(dx), ptr(dgate), ptr(dresidual),
                                   ptr(dweight), ptr(dscale), ptr(dnext), ptr(ws), ws.defined() ? ws_bytes : 0, stream_of(x)));
    return {dx, dweight, dgate, dresidual, dscale, dnext};
}

std::tuple<Tensor, Tensor, Tensor> norm_join_hip(const Tensor &x, const MaybeTensor &weight, const MaybeTensor &gate,
                                                 const MaybeTensor &residual, const MaybeTensor &scale,
                                                 const MaybeTensor &next_weight, double eps, int64_t activation, bool keep) {
    auto [out, next, stats] = norm_forward(x, or_undefined(weight), or_undefined(gate), or_undefined(residual), or_undefined(scale),
                                           or_undefined(next_weight), eps, activation, keep);
    if (!keep) stats = at::empty({0, x.numel() / x.size(-1)}, x.options().dtype(at::kFloat));
    return {out, or_empty(next, x), stats};
}

NormGradients norm_join_backward_hip(const MaybeTensor &grad_out, const MaybeTensor &grad_next, const Tensor &x,
                                     const MaybeTensor &weight, const MaybeTensor &gate, const MaybeTensor &residual,
                                     const MaybeTensor &scale, const MaybeTensor &next_weight, const Tensor &stats, double eps,
                                     int64_t activation) {
    return norm_backward(or_undefined(grad_out), or_undefined(grad_next), x, or_undefined(weight), or_undefined(gate),
                         or_undefined(residual), or_undefined(scale), or_undefined(next_weight), stats, eps, activation,
                         {true, true, true, true, true, true});
}

using NormOp = std::tuple<Tensor, Tensor, Tensor>(const Tensor &, const MaybeTensor &, const MaybeTensor &, const MaybeTensor &,
                                                  const MaybeTensor &, const MaybeTensor &, double, int64_t, bool);
using NormBackwardOp = NormGradients(const MaybeTensor &, const MaybeTensor &, const Tensor &, const MaybeTensor &,
                                     const MaybeTensor &, const MaybeTensor &, const MaybeTensor &, const MaybeTensor &,
                                     const Tensor &, double, int64_t);

template <bool DIRECT>
struct NormFunction : public torch::autograd::Function<NormFunction<DIRECT>> {
    static variable_list forward(AutogradContext *ctx, const Tensor &x, const MaybeTensor &maybe_weight,
                                 const MaybeTensor &maybe_gate, const MaybeTensor &maybe_residual, const MaybeTensor &maybe_scale,
                                 const MaybeTensor &maybe_next_weight, double eps, int64_t activation) {
        at::AutoDispatchBelowADInplaceOrView below;
        const Tensor weight = or_undefined(maybe_weight), gate = or_undefined(maybe_gate), residual = or_undefined(maybe_residual),
                     scale = or_undefined(maybe_scale), next_weight = or_undefined(maybe_next_weight);
        Tensor out, next, stats;
        if constexpr (DIRECT) {
            std::tie(out, next, stats) = norm_forward(x, weight, gate, residual, scale, next_weight, eps, activation, true);
        } else {
            static auto op = typed_op<NormOp>("pathsig::norm_join");
            std::tie(out, next, stats) = op.call(x, maybe_weight, maybe_gate, maybe_residual, maybe_scale, maybe_next_weight, eps,
                                                 activation, true);
        }
        // The residual is read again where the second norm's input is rebuilt.  Without that norm its gradient is the one from above,
        // and it may change after the call.
        ctx->save_for_backward({x, weight, gate, next_weight.defined() ? residual : Tensor(), scale, next_weight, stats});
        ctx->saved_data["residual"] = residual.defined();
        ctx->saved_data["eps"] = eps;
        ctx->saved_data["activation"] = activation;
        ctx->set_materialize_grads(false);
        if constexpr (DIRECT) {
            if (next_weight.defined()) return {out, next};
            return {out};
        }
        if (next_weight.defined())
            ctx->mark_non_differentiable({stats});
        else
            ctx->mark_non_differentiable({next, stats});
        return {out, next, stats};
    }
    static variable_list backward(AutogradContext *ctx, variable_list grads) {
        variable_list out(8);
        const Tensor &grad_out = grads[0], grad_next = grads.size() > 1 ? grads[1] : Tensor();
        if (!grad_out.defined() && !grad_next.defined()) return out;
        const auto s = ctx->get_saved_variables();
        const double eps = ctx->saved_data["eps"].toDouble();
        const int64_t activation = ctx->saved_data["activation"].toInt();
        bool direct = DIRECT && !at::GradMode::is_enabled();
        for (const Tensor &t : s) direct = direct && (!t.defined() || plain(t));
        for (const Tensor *t : {&grad_out, &grad_next}) direct = direct && (!t->defined() || plain(*t));
        const bool residual = ctx->saved_data["residual"].toBool();
        std::array<bool, 6> want{};
        for (int i = 0, present = 0; i < 6; ++i)  // (autograd counts the inputs that are there)
            want[i] = (i == 3 ? residual : s[i].defined()) && ctx->needs_input_grad(present++);
        if (want[3] && !s[3].defined() && std::count(want.begin(), want.end(), true) == 1) {
            out[3] = grad_out;
            return out;
        }
        NormGradients g;
        if (direct) {
            g = norm_backward(grad_out, grad_next, s[0], s[1], s[2], s[3], s[4], s[5], s[6], eps, activation, want);
        } else {
            static auto op = typed_op<NormBackwardOp>("pathsig::norm_join_backward");
            g = op.call(or_none(grad_out), or_none(grad_next), s[0], or_none(s[1]), or_none(s[2]), or_none(s[3]), or_none(s[4]),
                        or_none(s[5]), s[6], eps, activation);
        }
        const Tensor all[] = {std::get<0>(g), std::get<1>(g), std::get<2>(g), s[3].defined() ? std::get<3>(g) : grad_out, std::get<4>(g),
                              std::get<5>(g)};
        for (int i = 0; i < 6; ++i)
            if (want[i]) out[i] = all[i];
        return out;
    }
};

std::tuple<Tensor, Tensor, Tensor> norm_join_autograd(const Tensor &x, const MaybeTensor &weight, const MaybeTensor &gate,
                                                      const MaybeTensor &residual, const MaybeTensor &scale,
                                                      const MaybeTensor &next_weight, double eps, int64_t activation, bool keep) {
    const Tensor w = or_undefined(weight), g = or_undefined(gate), r = or_undefined(residual), s = or_undefined(scale),
                 n = or_undefined(next_weight);
    if (!any_grad({&x, &w, &g, &r, &s, &n})) {
        at::AutoDispatchBelowADInplaceOrView below;
        static auto op = typed_op<NormOp>("pathsig::norm_join");
        return op.call(x, weight, gate, residual, scale, next_weight, eps, activation, keep);
    }
    auto out = NormFunction<false>::apply(x, weight, gate, residual, scale, next_weight, eps, activation);
    return {out[0], out[1], out[2]};
}

// ---- arguments of the functions of the extension ------------------------------------------------------------------
// a plain CUDA tensor, or (optional) None
bool plain_arg(PyObject *obj, Tensor &out, bool optional) {
    if (optional && obj == Py_None) return true;
    return tensor_arg(obj, out) && plain(out);
}

PyObject *wrap_pair(Tensor first, Tensor second) {
    PyObject *pair = PyTuple_New(2);
    if (!pair) return nullptr;
    PyTuple_SET_ITEM(pair, 0, THPVariable_Wrap(std::move(first)));
    PyTuple_SET_ITEM(pair, 1, THPVariable_Wrap(std::move(second)));
    return pair;
}

}  // namespace

// All arguments positional; None when the call is not one for this way.
// (q, k, v, log_decay, state, lengths, scale, return_state)
PyObject *py_linear_attention(PyObject *, PyObject *const *args, Py_ssize_t nargs) {
    HANDLE_TH_ERRORS
    Tensor t[6], out, last;
    if (nargs != 8 || !PyFloat_Check(args[6])) Py_RETURN_NONE;
    for (int i = 0; i < 6; ++i)
        if (!plain_arg(args[i], t[i], i >= 4)) Py_RETURN_NONE;
    const double scale = PyFloat_AS_DOUBLE(args[6]);
    const bool return_state = args[7] == Py_True;
    {
        pybind11::gil_scoped_release no_gil;
        if (any_grad({&t[0], &t[1], &t[2], &t[3], &t[4]})) {
            auto both = AttentionFunction<true>::apply(t[0], t[1], t[2], t[3], or_none(t[4]), or_none(t[5]), scale, return_state);
            out = both[0];
            if (return_state) last = both[1];
        } else {
            at::AutoDispatchBelowADInplaceOrView below;
            Tensor kept;
            std::tie(out, last, kept) = attention_forward(t[0], t[1], t[2], t[3], t[4], t[5], scale, return_state, false);
        }
    }
    if (!return_state) return THPVariable_Wrap(std::move(out));
    return wrap_pair(std::move(out), std::move(last));
    END_HANDLE_TH_ERRORS
}

// (q, k, v, log_decay, state, scale)
PyObject *py_linear_attention_step(PyObject *, PyObject *const *args, Py_ssize_t nargs) {
    HANDLE_TH_ERRORS
    Tensor t[5], out;
    if (nargs != 6 || !PyFloat_Check(args[5])) Py_RETURN_NONE;
    for (int i = 0; i < 5; ++i)
        if (!plain_arg(args[i], t[i], false)) Py_RETURN_NONE;
    if (any_grad({&t[0], &t[1], &t[2], &t[3], &t[4]})) Py_RETURN_NONE;  // the operator refuses it
    const double scale = PyFloat_AS_DOUBLE(args[5]);
    {
        pybind11::gil_scoped_release no_gil;
        at::AutoDispatchBelowADInplaceOrView below;
        out = attention_step(t[0], t[1], t[2], t[3], t[4], scale);
    }
    return THPVariable_Wrap(std::move(out));
    END_HANDLE_TH_ERRORS
}

// (x, weight, gate, residual, scale, next_weight, eps, activation)
PyObject *py_norm_join(PyObject *, PyObject *const *args, Py_ssize_t nargs) {
    HANDLE_TH_ERRORS
    Tensor t[6], out, next;
    if (nargs != 8 || !PyFloat_Check(args[6]) || !PyLong_Check(args[7])) Py_RETURN_NONE;
    for (int i = 0; i < 6; ++i)
        if (!plain_arg(args[i], t[i], i >= 1)) Py_RETURN_NONE;
    const double eps = PyFloat_AS_DOUBLE(args[6]);
    const int64_t activation = PyLong_AsLongLong(args[7]);
    {
        pybind11::gil_scoped_release no_gil;
        if (any_grad({&t[0], &t[1], &t[2], &t[3], &t[4], &t[5]})) {
            auto all = NormFunction<true>::apply(t[0], or_none(t[1]), or_none(t[2]), or_none(t[3]), or_none(t[4]), or_none(t[5]), eps,
                                                 activation);
            out = all[0];
            if (t[5].defined()) next = all[1];
        } else {
            at::AutoDispatchBelowADInplaceOrView below;
            Tensor stats;
            std::tie(out, next, stats) = norm_forward(t[0], t[1], t[2], t[3], t[4], t[5], eps, activation, false);
        }
    }
    if (!t[5].defined()) return THPVariable_Wrap(std::move(out));
    return wrap_pair(std::move(out), std::move(next));
    END_HANDLE_TH_ERRORS
}

}  // namespace psig_torch

TORCH_LIBRARY_FRAGMENT(pathsig, m) {
    const std::vector<at::Tag> pt2{at::Tag::pt2_compliant_tag};
    m.def("linear_attention(Tensor q, Tensor k, Tensor v, Tensor log_decay, Tensor? state, Tensor? lengths, float scale, "
          "bool return_state) -> (Tensor, Tensor)", pt2);
    m.def("linear_attention_backward(Tensor grad_out, Tensor? grad_state, Tensor q, Tensor k, Tensor v, Tensor log_decay, "
          "Tensor? state, Tensor? lengths, float scale, bool want_log_decay, bool want_state) "
          "-> (Tensor, Tensor, Tensor, Tensor, Tensor)", pt2);
    m.def("linear_attention_step(Tensor q, Tensor k, Tensor v, Tensor log_decay, Tensor(a!) state, float scale) -> Tensor", pt2);
    m.def("norm_join(Tensor x, Tensor? weight, Tensor? gate, Tensor? residual, Tensor? scale, Tensor? next_weight, float eps, "
          "int activation, bool keep) -> (Tensor, Tensor, Tensor)", pt2);
    m.def("norm_join_backward(Tensor? grad_out, Tensor? grad_next, Tensor x, Tensor? weight, Tensor? gate, Tensor? residual, "
          "Tensor? scale, Tensor? next_weight, Tensor statistics, float eps, int activation) "
          "-> (Tensor, Tensor, Tensor, Tensor, Tensor, Tensor)", pt2);
}

TORCH_LIBRARY_IMPL(pathsig, CUDA, m) {
    m.impl("linear_attention", &psig_torch::linear_attention_hip);
    m.impl("linear_attention_backward", &psig_torch::linear_attention_backward_hip);
    m.impl("linear_attention_step", &psig_torch::linear_attention_step_hip);
    m.impl("norm_join", &psig_torch::norm_join_hip);
    m.impl("norm_join_backward", &psig_torch::norm_join_backward_hip);
}

TORCH_LIBRARY_IMPL(pathsig, Autograd, m) {
    m.impl("linear_attention", &psig_torch::linear_attention_autograd);
    m.impl("linear_attention_step", &psig_torch::linear_attention_step_autograd);
    m.impl("norm_join", &psig_torch::norm_join_autograd);
    // (without these, a gradient of a gradient would go on without their part of it, with a warning alone)
    m.impl("linear_attention_backward", torch::autograd::autogradNotImplementedFallback());
    m.impl("norm_join_backward", torch::autograd::autogradNotImplementedFallback());
}
