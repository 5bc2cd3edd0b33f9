// The output head's operators on torch tensors: allocation, the C-ABI call on the tensors' current stream, and the autograd
// nodes. In C++ for the host's time: a training step's backward pass runs on autograd's own thread, where a node in Python waits
// for the interpreter lock (a step of 16 rows 96 us with Python nodes, 52 with these), and a call's allocations are most of its
// cost (one row's log-probabilities 12.6 us from Python, 6.5 from here). Arguments
// are checked by yggdrasil_amd/ops.py, those of plain calls here; the library's entries come as addresses, so that there is one copy of it.
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/extension.h>

#include <map>
#include <optional>
#include <string>

#include "../../include/ygg_hip.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
typedef std::optional<Tensor> Maybe;

struct {
    decltype(&ygg_logprobs_scratch) logprobs_scratch;
    decltype(&ygg_logprobs) logprobs;
    decltype(&ygg_logprobs_grad) logprobs_grad;
    decltype(&ygg_grouped_matmul) grouped_matmul;
    decltype(&ygg_grouped_grad_x) grouped_grad_x;
    decltype(&ygg_grouped_grad_w) grouped_grad_w;
    decltype(&ygg_int8_scratch) int8_scratch;
    decltype(&ygg_int8_linear) int8_linear;
    decltype(&ygg_last_error) last_error;
} api;

void bind(const std::map<std::string, uintptr_t> &at) {
    auto set = [&](auto &f, const char *name) { f = (std::decay_t<decltype(f)>)at.at(name); };
    set(api.logprobs_scratch, "ygg_logprobs_scratch");
    set(api.logprobs, "ygg_logprobs");
    set(api.logprobs_grad, "ygg_logprobs_grad");
    set(api.grouped_matmul, "ygg_grouped_matmul");
    set(api.grouped_grad_x, "ygg_grouped_grad_x");
    set(api.grouped_grad_w, "ygg_grouped_grad_w");
    set(api.int8_scratch, "ygg_int8_scratch");
    set(api.int8_linear, "ygg_int8_linear");
    set(api.last_error, "ygg_last_error");
}

void check(int rc) {
    if (rc) throw std::runtime_error(std::string(api.last_error()) + " (error " + std::to_string(rc) + ")");
}
int type_of(const Tensor &t) { return t.scalar_type() == at::kFloat ? 0 : t.scalar_type() == at::kBFloat16 ? 1 : 2; }
void *stream_of(const Tensor &t) { return c10::hip::getCurrentHIPStream(t.get_device()).stream(); }
template <class T = void> T *ptr(const Tensor &t) { return t.defined() ? (T *)t.data_ptr() : nullptr; }
Tensor empty(const Tensor &like, at::IntArrayRef size, at::ScalarType type) { return at::empty(size, like.options().dtype(type)); }
// Forward-mode derivatives are refused: there are none here, and a tangent that is left out would count as zero. A tensor that
// has one need not require a gradient.
void no_tangents(const char *name, std::initializer_list<Tensor> tensors) {
    if (!c10::AutogradState::get_tls_state().get_fw_grad_mode()) return;
    for (const Tensor &t : tensors)
        if (t.defined() && t._fw_grad(0).defined()) throw std::runtime_error(std::string(name) + " has no forward-mode derivative");
}
// gradients of gradients are refused where they are asked for, not when a graph is only kept
variable_list once(variable_list grads, const char *name) {
    if (!at::GradMode::is_enabled()) return grads;
    for (Tensor &g : grads) g.set_requires_grad(true);     // new tensors, of which it makes outputs that refuse
    auto refuse = std::make_shared<torch::autograd::DelayedError>(std::string(name) + " has no second derivative", grads.size());
    return (*refuse)(std::move(grads));
}

struct LogProbs {
    Tensor logp, entropy, top_logp, top_ids, stats;
};
LogProbs logprobs(const Tensor &x, const Tensor &targets, int64_t top, bool keep) {
    const c10::DeviceGuard guard(x.device());
    const int64_t rows = x.size(0), V = x.size(1);
    LogProbs r;
    if (targets.defined()) r.logp = empty(x, {rows}, at::kFloat);
    r.entropy = empty(x, {rows}, at::kFloat);
    if (top) {
        r.top_logp = empty(x, {rows, top}, at::kFloat);
        r.top_ids = empty(x, {rows, top}, at::kInt);
    }
    if (keep) r.stats = empty(x, {rows, 2}, at::kFloat);
    const int64_t need = rows ? api.logprobs_scratch(type_of(x), rows, V, top) : 0;
    Tensor scratch;
    if (need) scratch = empty(x, {need}, at::kByte);
    check(api.logprobs(x.data_ptr(), type_of(x), rows, V, rows > 1 ? x.stride(0) : V, ptr(targets),
                       targets.defined() ? targets.element_size() : 0, top, ptr<float>(r.logp), ptr<float>(r.entropy),
                       ptr<float>(r.top_logp), ptr<int32_t>(r.top_ids), ptr<float>(r.stats), ptr(scratch), need, stream_of(x)));
    return r;
}
struct TokenLogprobs : torch::autograd::Function<TokenLogprobs> {
    // outputs: the entropy, the log-probabilities if there are targets, the alternatives' and their ids if there are any
    static variable_list forward(AutogradContext *ctx, const Tensor &x, const Maybe &targets, int64_t top) {
        at::AutoDispatchBelowADInplaceOrView guard;
        const Tensor t = targets.value_or(Tensor());
        LogProbs r = logprobs(x, t, top, true);
        ctx->save_for_backward({x, t, r.entropy, r.top_ids, r.stats});
        ctx->set_materialize_grads(false);
        variable_list out{r.entropy};
        if (t.defined()) out.push_back(r.logp);
        if (top) {
            ctx->mark_non_differentiable({r.top_ids});
            out.push_back(r.top_logp);
            out.push_back(r.top_ids);
        }
        return out;
    }
    static variable_list backward(AutogradContext *ctx, variable_list grads) {
        const variable_list s = ctx->get_saved_variables();
        const Tensor &x = s[0], &t = s[1], &entropy = s[2], &top_ids = s[3], &stats = s[4];
        const c10::DeviceGuard guard(x.device());
        Tensor dx;
        {
            const at::AutoGradMode none(false);
            auto f32 = [](const Tensor &g) { return g.defined() ? g.to(at::kFloat).contiguous() : g; };
            const int at_logp = t.defined(), at_top = at_logp + 1;
            for (const Tensor &g : grads) no_tangents("token_logprobs' gradient", {g});
            const Tensor ge = f32(grads[0]), gl = at_logp ? f32(grads[1]) : Tensor(), gt = top_ids.defined() ? f32(grads[at_top]) : Tensor();
            const int64_t rows = x.size(0), V = x.size(1);
            dx = empty(x, {rows, V}, x.scalar_type());
            check(api.logprobs_grad(x.data_ptr(), type_of(x), rows, V, rows > 1 ? x.stride(0) : V, ptr(t),
                                    t.defined() ? t.element_size() : 0, top_ids.defined() ? top_ids.size(1) : 0, ptr<float>(entropy),
                                    ptr<int32_t>(top_ids), ptr<float>(stats), ptr<float>(gl), ptr<float>(ge), ptr<float>(gt), ptr(dx),
                                    stream_of(x)));
        }
        return {once({dx}, "token_logprobs")[0], Tensor(), Tensor()};
    }
};
// logp, entropy, top_logp, top_ids; None where there are none
std::tuple<Maybe, Tensor, Maybe, Maybe> token_logprobs(const Tensor &x, const Maybe &targets, int64_t top) {
    no_tangents("token_logprobs", {x});
    auto some = [](const Tensor &t) { return t.defined() ? Maybe(t) : Maybe(); };
    if (x.requires_grad() && at::GradMode::is_enabled()) {
        const variable_list r = TokenLogprobs::apply(x, targets, top);
        const size_t n = targets.has_value();
        return {n ? Maybe(r[1]) : Maybe(), r[0], top ? Maybe(r[n + 1]) : Maybe(), top ? Maybe(r[n + 2]) : Maybe()};
    }
    const LogProbs r = logprobs(x, targets.value_or(Tensor()), top, false);
    return {some(r.logp), r.entropy, some(r.top_logp), some(r.top_ids)};
}

// fn of a (rows), b (the matrices or rows) into a tensor of out_size; shape: w's
template <class F>
Tensor grouped(F fn, const Tensor &a, const Tensor &b, const Tensor &offsets, const Tensor &order, int64_t M, at::IntArrayRef shape,
               at::IntArrayRef out_size) {
    const c10::DeviceGuard guard(a.device());
    Tensor out = empty(a, out_size, a.scalar_type());
    check(fn(a.data_ptr(), b.data_ptr(), type_of(a), ptr<int32_t>(offsets), ptr<int32_t>(order), M, shape[0], shape[1], shape[2],
             out.data_ptr(), stream_of(a)));
    return out;
}
struct GroupedMatmul : torch::autograd::Function<GroupedMatmul> {
    static Tensor forward(AutogradContext *ctx, const Tensor &x, const Tensor &w, const Tensor &offsets, const Maybe &order) {
        at::AutoDispatchBelowADInplaceOrView guard;
        const Tensor o = order.value_or(Tensor());
        ctx->save_for_backward({x, w, offsets, o});
        return grouped(api.grouped_matmul, x, w, offsets, o, x.size(0), w.sizes(), {x.size(0), w.size(1)});
    }
    static variable_list backward(AutogradContext *ctx, variable_list grads) {
        const variable_list s = ctx->get_saved_variables();
        const Tensor &x = s[0], &w = s[1], &offsets = s[2], &order = s[3];
        const bool to_x = ctx->needs_input_grad(0), to_w = ctx->needs_input_grad(1);
        variable_list out;
        {
            const at::AutoGradMode none(false);
            no_tangents("grouped_matmul's gradient", {grads[0]});
            const Tensor dy = grads[0].contiguous();
            if (to_x) out.push_back(grouped(api.grouped_grad_x, dy, w, offsets, order, x.size(0), w.sizes(), x.sizes()));
            if (to_w) out.push_back(grouped(api.grouped_grad_w, dy, x, offsets, order, x.size(0), w.sizes(), w.sizes()));
        }
        out = once(std::move(out), "grouped_matmul");
        return {to_x ? out[0] : Tensor(), to_w ? out[to_x] : Tensor(), Tensor(), Tensor()};
    }
};
Tensor grouped_matmul(const Tensor &x, const Tensor &w, const Tensor &offsets, const Maybe &order) {
    no_tangents("grouped_matmul", {x, w});
    if ((x.requires_grad() || w.requires_grad()) && at::GradMode::is_enabled()) return GroupedMatmul::apply(x, w, offsets, order);
    return grouped(api.grouped_matmul, x, w, offsets, order.value_or(Tensor()), x.size(0), w.sizes(), {x.size(0), w.size(1)});
}

Tensor int8_linear(const Tensor &x, const Tensor &w, const Tensor &w_scale) {
    no_tangents("int8_linear", {x, w_scale});
    const c10::DeviceGuard guard(x.device());
    const int64_t M = x.size(0), K = x.size(1), N = w.size(0);
    Tensor y = empty(x, {M, N}, x.scalar_type());
    const int64_t need = M ? api.int8_scratch(M, N, K) : 0;
    Tensor scratch;
    if (need) scratch = empty(x, {need}, at::kByte);
    check(api.int8_linear(x.data_ptr(), type_of(x), ptr<int8_t>(w), ptr<float>(w_scale), M, N, K, y.data_ptr(), ptr(scratch), need,
                          stream_of(x)));
    return y;
}

// The calls on tensors that need no reshaping, checked here; nothing where they do, or where a check fails and ops.py says why
bool floats(const Tensor &t, int64_t dim) {
    const auto d = t.scalar_type();
    return t.is_cuda() && (d == at::kFloat || d == at::kBFloat16 || d == at::kHalf) && t.dim() == dim && t.is_contiguous();
}
bool like(const Tensor &t, const Tensor &other, at::ScalarType type, int64_t dim) {
    return t.device() == other.device() && t.scalar_type() == type && t.dim() == dim && t.is_contiguous();
}
bool within(int64_t v, int64_t lo, int64_t hi) { return v >= lo && v <= hi; }

std::optional<std::tuple<Maybe, Tensor, Maybe, Maybe>> plain_token_logprobs(const Tensor &x, const Maybe &targets, int64_t top) {
    if (!floats(x, 2) || !within(x.size(1), 1, YGG_MOST_VOCAB) || !within(top, 0, YGG_MOST_TOP)) return std::nullopt;
    if (targets && !((like(*targets, x, at::kInt, 1) || like(*targets, x, at::kLong, 1)) && targets->size(0) == x.size(0)))
        return std::nullopt;
    return token_logprobs(x, targets, top);
}
Maybe plain_grouped_matmul(const Tensor &x, const Tensor &w, const Tensor &offsets, const Maybe &order) {
    if (!floats(x, 2) || !like(w, x, x.scalar_type(), 3) || w.size(2) != x.size(1) || x.size(0) > YGG_MOST_ROWS ||
        !within(w.size(0), 1, YGG_MOST_EXPERTS) || !within(w.size(1), 1, YGG_MOST_INNER) || !within(w.size(2), 1, YGG_MOST_INNER) ||
        !like(offsets, x, at::kInt, 1) || offsets.size(0) != w.size(0) + 1)
        return std::nullopt;
    if (order && !(like(*order, x, at::kInt, 1) && order->size(0) == x.size(0))) return std::nullopt;
    return grouped_matmul(x, w, offsets, order);
}
Maybe plain_int8_linear(const Tensor &x, const Tensor &w, const Tensor &w_scale) {
    if (!floats(x, 2) || ((x.requires_grad() || w_scale.requires_grad()) && at::GradMode::is_enabled()) ||
        !like(w, x, at::kChar, 2) || w.size(1) != x.size(1) || x.size(0) > YGG_MOST_ROWS ||
        !within(w.size(0), 1, YGG_MOST_VOCAB) || !within(w.size(1), 1, YGG_MOST_INNER) ||
        !like(w_scale, x, at::kFloat, 1) || w_scale.size(0) != w.size(0))
        return std::nullopt;
    return int8_linear(x, w, w_scale);
}

}  // namespace

PYBIND11_MODULE(_ygg_torch, m) {
    m.def("bind", &bind);
    m.def("token_logprobs", &token_logprobs);
    m.def("grouped_matmul", &grouped_matmul);
    m.def("int8_linear", &int8_linear);
    m.def("plain_token_logprobs", &plain_token_logprobs);
    m.def("plain_grouped_matmul", &plain_grouped_matmul);
    m.def("plain_int8_linear", &plain_int8_linear);
}
