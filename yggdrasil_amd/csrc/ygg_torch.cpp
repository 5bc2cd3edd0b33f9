// The operators of an output head and of a recurrent block on torch tensors: allocation, the C-ABI call on the tensors' current stream, and the autograd
// nodes. In C++ for the host's time: a training step's backward pass runs on autograd's own thread, where a node in Python waits
// for the interpreter lock (a step of 16 rows 96 us with Python nodes, 52 with these), and a call's allocations are most of its
// cost (one row's log-probabilities 12.6 us from Python, 6.5 from here). Arguments
// are checked by yggdrasil_amd/ops.py, those of plain calls here; the library's entries come as addresses, so that there is one copy of it.
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/extension.h>

#include <algorithm>
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
    decltype(&ygg_layer_norm) layer_norm;
    decltype(&ygg_layer_norm_scratch) layer_norm_scratch;
    decltype(&ygg_layer_norm_grad) layer_norm_grad;
    decltype(&ygg_gated_scan) gated_scan;
    decltype(&ygg_gated_scan_scratch) gated_scan_scratch;
    decltype(&ygg_gated_scan_kept) gated_scan_kept;
    decltype(&ygg_gated_scan_grad) gated_scan_grad;
    decltype(&ygg_gated_linear) gated_linear;
    decltype(&ygg_gated_linear_kept) gated_linear_kept;
    decltype(&ygg_gated_linear_scratch) gated_linear_scratch;
    decltype(&ygg_gated_linear_grad) gated_linear_grad;
    decltype(&ygg_clip_scratch) clip_scratch;
    decltype(&ygg_clip_grad_norm) clip_grad_norm;
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
    set(api.layer_norm, "ygg_layer_norm");
    set(api.layer_norm_scratch, "ygg_layer_norm_scratch");
    set(api.layer_norm_grad, "ygg_layer_norm_grad");
    set(api.gated_scan, "ygg_gated_scan");
    set(api.gated_scan_scratch, "ygg_gated_scan_scratch");
    set(api.gated_scan_kept, "ygg_gated_scan_kept");
    set(api.gated_scan_grad, "ygg_gated_scan_grad");
    set(api.gated_linear, "ygg_gated_linear");
    set(api.gated_linear_kept, "ygg_gated_linear_kept");
    set(api.gated_linear_scratch, "ygg_gated_linear_scratch");
    set(api.gated_linear_grad, "ygg_gated_linear_grad");
    set(api.clip_scratch, "ygg_clip_scratch");
    set(api.clip_grad_norm, "ygg_clip_grad_norm");
    set(api.last_error, "ygg_last_error");
}

void check(int rc) {
    if (rc) throw std::runtime_error(std::string(api.last_error()) + " (error " + std::to_string(rc) + ")");
}
int type_of(at::ScalarType t) { return t == at::kFloat ? 0 : t == at::kBFloat16 ? 1 : 2; }
int type_of(const Tensor &t) { return type_of(t.scalar_type()); }
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

// ---------------------------------------------------------------------------------------------- a recurrent block's operators
Tensor scratch_of(const Tensor &like, int64_t bytes) { return bytes ? empty(like, {bytes}, at::kByte) : Tensor(); }
Tensor or_none(const Maybe &t) { return t.value_or(Tensor()); }
bool wants_grad(std::initializer_list<Tensor> tensors) {
    if (!at::GradMode::is_enabled()) return false;
    for (const Tensor &t : tensors)
        if (t.defined() && t.requires_grad()) return true;
    return false;
}
// which of the tensors that a node got (undefined ones are none of its inputs) a backward pass wants gradients of
std::vector<bool> wanted(AutogradContext *ctx, std::initializer_list<bool> given) {
    std::vector<bool> want;
    size_t edge = 0;
    for (bool g : given) want.push_back(g && ctx->needs_input_grad(edge++));
    return want;
}

// rows (M, n) any distance apart -> y, and a row's mean and inverse deviation if they are kept
std::pair<Tensor, Tensor> layer_norm_of(const Tensor &x, const Tensor &w, const Tensor &b, double eps, bool keep) {
    const c10::DeviceGuard guard(x.device());
    const int64_t rows = x.size(0), n = x.size(1);
    Tensor y = empty(x, {rows, n}, x.scalar_type()), stats;
    if (keep) stats = empty(x, {rows, 2}, at::kFloat);
    const Tensor &any = w.defined() ? w : b;
    check(api.layer_norm(x.data_ptr(), type_of(x), rows, n, rows > 1 ? x.stride(0) : n, ptr(w), ptr(b), any.defined() ? type_of(any) : 0,
                         eps, y.data_ptr(), ptr<float>(stats), stream_of(x)));
    return {y, stats};
}
struct LayerNorm : torch::autograd::Function<LayerNorm> {
    static Tensor forward(AutogradContext *ctx, const Tensor &x, const Maybe &w, const Maybe &b, double eps) {
        at::AutoDispatchBelowADInplaceOrView guard;
        auto [y, stats] = layer_norm_of(x, or_none(w), or_none(b), eps, true);
        ctx->save_for_backward({x, or_none(w), stats});
        ctx->saved_data["type"] = w ? (int64_t)type_of(*w) : b ? (int64_t)type_of(*b) : 0;
        ctx->saved_data["w"] = w.has_value();
        ctx->saved_data["b"] = b.has_value();
        return y;
    }
    static variable_list backward(AutogradContext *ctx, variable_list grads) {
        const variable_list s = ctx->get_saved_variables();
        const Tensor &x = s[0], &w = s[1], &stats = s[2];
        const std::vector<bool> want = wanted(ctx, {true, ctx->saved_data["w"].toBool(), ctx->saved_data["b"].toBool()});
        const c10::DeviceGuard guard(x.device());
        variable_list out(3), made;
        {
            const at::AutoGradMode none(false);
            no_tangents("layer_norm's gradient", {grads[0]});
            const Tensor dy = grads[0].contiguous();
            const int64_t rows = x.size(0), n = x.size(1), type = ctx->saved_data["type"].toInt();
            const at::ScalarType kind = type == 0 ? at::kFloat : x.scalar_type();
            if (want[0]) out[0] = empty(x, {rows, n}, x.scalar_type());
            for (int k : {1, 2})
                if (want[k]) out[k] = empty(x, {n}, kind);
            const int64_t need = want[1] || want[2] || n > 16384 ? api.layer_norm_scratch(type_of(x), rows, n) : 0;
            const Tensor scratch = scratch_of(x, need);
            check(api.layer_norm_grad(x.data_ptr(), type_of(x), rows, n, rows > 1 ? x.stride(0) : n, ptr(w), type, ptr<float>(stats),
                                      dy.data_ptr(), ptr(out[0]), ptr(out[1]), ptr(out[2]), ptr(scratch), need, stream_of(x)));
            for (const Tensor &t : out)
                if (t.defined()) made.push_back(t);
        }
        made = once(std::move(made), "layer_norm");
        size_t k = 0;
        for (Tensor &t : out)
            if (t.defined()) t = made[k++];
        out.push_back(Tensor());
        return out;
    }
};
Tensor layer_norm(const Tensor &x, const Maybe &w, const Maybe &b, double eps) {
    no_tangents("layer_norm", {x, or_none(w), or_none(b)});
    if (wants_grad({x, or_none(w), or_none(b)})) return LayerNorm::apply(x, w, b, eps);
    return layer_norm_of(x, or_none(w), or_none(b), eps, false).first;
}

// gate, x (B, T, n), a step's channels next to each other; state (B, n) or undefined -> h, the last state, and
// what the gate's gradient wants if it is kept
std::tuple<Tensor, Tensor, Tensor> gated_scan_of(const Tensor &gate, const Tensor &x, const Tensor &state, bool keep) {
    const c10::DeviceGuard guard(x.device());
    const int64_t B = x.size(0), T = x.size(1), n = x.size(2);
    Tensor h = empty(x, {B, T, n}, x.scalar_type()), last = empty(x, {B, n}, at::kFloat), kept;
    if (keep) kept = scratch_of(x, api.gated_scan_kept(B, T, n));
    const int64_t need = api.gated_scan_scratch(type_of(x), type_of(gate), B, T, n);
    const Tensor scratch = scratch_of(x, need);
    check(api.gated_scan(gate.data_ptr(), type_of(gate), gate.stride(0), gate.stride(1), x.data_ptr(), type_of(x), x.stride(0), x.stride(1),
                         B, T, n, ptr<float>(state), h.data_ptr(), ptr<float>(last), ptr<float>(kept), ptr(scratch), need, stream_of(x)));
    return {h, last, kept};
}
struct GatedScan : torch::autograd::Function<GatedScan> {
    static variable_list forward(AutogradContext *ctx, const Tensor &gate, const Tensor &x, const Maybe &state) {
        at::AutoDispatchBelowADInplaceOrView guard;
        const bool keep = gate.requires_grad();
        auto [h, last, kept] = gated_scan_of(gate, x, or_none(state), keep);
        ctx->save_for_backward({gate, keep ? x : Tensor(), keep ? or_none(state) : Tensor(), kept});
        ctx->saved_data["type"] = (int64_t)x.scalar_type();
        ctx->saved_data["state"] = state.has_value();
        ctx->set_materialize_grads(false);
        return {h, last};
    }
    static variable_list backward(AutogradContext *ctx, variable_list grads) {
        const variable_list s = ctx->get_saved_variables();
        const Tensor &gate = s[0], &x = s[1], &state = s[2], &kept = s[3];
        const at::ScalarType type = (at::ScalarType)ctx->saved_data["type"].toInt();
        const std::vector<bool> want = wanted(ctx, {true, true, ctx->saved_data["state"].toBool()});
        const c10::DeviceGuard guard(gate.device());
        variable_list out(3), made;
        {
            const at::AutoGradMode none(false);
            for (const Tensor &g : grads) no_tangents("gated_scan's gradient", {g});
            const Tensor dh = grads[0].defined() ? grads[0].contiguous() : Tensor(), dlast = grads[1].defined() ? grads[1].contiguous() : Tensor();
            const int64_t B = gate.size(0), T = gate.size(1), n = gate.size(2);
            if (want[0]) out[0] = empty(gate, {B, T, n}, gate.scalar_type());
            if (want[1]) out[1] = empty(gate, {B, T, n}, type);
            if (want[2]) out[2] = empty(gate, {B, n}, at::kFloat);
            const int64_t need = api.gated_scan_scratch(type_of(type), type_of(gate), B, T, n);
            const Tensor scratch = scratch_of(gate, need);
            check(api.gated_scan_grad(gate.data_ptr(), type_of(gate), gate.stride(0), gate.stride(1), ptr(x), type_of(type),
                                      x.defined() ? x.stride(0) : 0, x.defined() ? x.stride(1) : 0, B, T, n, ptr<float>(state),
                                      ptr<float>(kept), ptr(dh), ptr<float>(dlast), ptr(out[1]), ptr(out[0]), ptr<float>(out[2]),
                                      ptr(scratch), need, stream_of(gate)));
            for (const Tensor &t : out)
                if (t.defined()) made.push_back(t);
        }
        made = once(std::move(made), "gated_scan");
        size_t k = 0;
        for (Tensor &t : out)
            if (t.defined()) t = made[k++];
        return out;
    }
};
std::pair<Tensor, Tensor> gated_scan(const Tensor &gate, const Tensor &x, const Maybe &state) {
    no_tangents("gated_scan", {gate, x, or_none(state)});
    if (wants_grad({gate, x, or_none(state)})) {
        const variable_list r = GatedScan::apply(gate, x, state);
        return {r[0], r[1]};
    }
    auto [h, last, kept] = gated_scan_of(gate, x, or_none(state), false);
    return {h, last};
}

// x (M, K), w (2, N, K) -> y, and g and u if they are kept
std::pair<Tensor, Tensor> gated_linear_of(const Tensor &x, const Tensor &w, int64_t act, bool keep) {
    const c10::DeviceGuard guard(x.device());
    const int64_t M = x.size(0), N = w.size(1), K = x.size(1);
    Tensor y = empty(x, {M, N}, x.scalar_type()), gu;
    if (keep) gu = empty(x, {api.gated_linear_kept(type_of(x), M, N)}, at::kByte);
    check(api.gated_linear(x.data_ptr(), w.data_ptr(), type_of(x), act, M, N, K, y.data_ptr(), ptr(gu), stream_of(x)));
    return {y, gu};
}
struct GatedLinear : torch::autograd::Function<GatedLinear> {
    static Tensor forward(AutogradContext *ctx, const Tensor &x, const Tensor &w, int64_t act) {
        at::AutoDispatchBelowADInplaceOrView guard;
        auto [y, gu] = gated_linear_of(x, w, act, true);
        ctx->save_for_backward({x, w, gu});
        ctx->saved_data["act"] = act;
        return y;
    }
    static variable_list backward(AutogradContext *ctx, variable_list grads) {
        const variable_list s = ctx->get_saved_variables();
        const Tensor &x = s[0], &w = s[1], &gu = s[2];
        const bool to_x = ctx->needs_input_grad(0), to_w = ctx->needs_input_grad(1);
        const c10::DeviceGuard guard(x.device());
        variable_list out;
        {
            const at::AutoGradMode none(false);
            no_tangents("gated_linear's gradient", {grads[0]});
            const Tensor dy = grads[0].contiguous();
            const int64_t M = x.size(0), N = w.size(1), K = x.size(1), need = api.gated_linear_scratch(type_of(x), M, N, K);
            const Tensor scratch = scratch_of(x, need);
            if (to_x) out.push_back(empty(x, {M, K}, x.scalar_type()));
            if (to_w) out.push_back(empty(x, {2, N, K}, x.scalar_type()));
            check(api.gated_linear_grad(x.data_ptr(), w.data_ptr(), gu.data_ptr(), dy.data_ptr(), type_of(x), ctx->saved_data["act"].toInt(),
                                        M, N, K, to_x ? out[0].data_ptr() : nullptr, to_w ? out[to_x].data_ptr() : nullptr, ptr(scratch),
                                        need, stream_of(x)));
        }
        out = once(std::move(out), "gated_linear");
        return {to_x ? out[0] : Tensor(), to_w ? out[to_x] : Tensor(), Tensor()};
    }
};
Tensor gated_linear(const Tensor &x, const Tensor &w, int64_t act) {
    no_tangents("gated_linear", {x, w});
    if (wants_grad({x, w})) return GatedLinear::apply(x, w, act);
    return gated_linear_of(x, w, act, false).first;
}

// The norm of the tensors' values together and, with clip, the tensors times min(1, most / norm): into out, tensors of their
// sizes and types (themselves among them), or new ones. Memory that is written may be no other tensor's.
struct Range {
    uintptr_t from, end;
    size_t i;
};
std::vector<Range> ranges_of(const std::vector<Tensor> &tensors) {
    std::vector<Range> r;
    for (size_t i = 0; i < tensors.size(); i++) {
        const uintptr_t p = (uintptr_t)tensors[i].data_ptr();
        if (tensors[i].numel()) r.push_back({p, p + tensors[i].nbytes(), i});
    }
    return r;
}
std::pair<std::vector<Tensor>, Tensor> clip_grad_norm(std::vector<Tensor> in, double most, bool clip, const std::optional<std::vector<Tensor>> &to) {
    const Tensor first = in.at(0);
    for (const Tensor &t : in) no_tangents("clip_grad_norm", {t});
    const c10::DeviceGuard guard(first.device());
    const at::AutoGradMode none(false);
    at::AutoDispatchBelowADInplaceOrView below;      // for the time of many allocations
    std::vector<Tensor> out;
    if (clip && to) {
        out = *to;
        for (const Tensor &t : out)
            if (t.layout() != at::kStrided || !t.is_non_overlapping_and_dense()) throw py::value_error("out must hold dense tensors");
    }
    std::vector<const void *> from(in.size());
    std::vector<void *> into(in.size());
    std::vector<int64_t> sizes(in.size());
    std::vector<int> types(in.size());
    for (size_t i = 0; i < in.size(); i++) {
        // values go in the order they lie in memory, the same in both
        if (!in[i].is_non_overlapping_and_dense()) in[i] = in[i].contiguous();
        if (clip) {
            if (!to) out.push_back(at::empty_strided(in[i].sizes(), in[i].strides(), in[i].options()));
            if (out[i].strides() != in[i].strides()) in[i] = at::empty_like(out[i]).copy_(in[i]);
            into[i] = out[i].data_ptr();
        }
        from[i] = in[i].data_ptr();
        sizes[i] = in[i].numel();
        types[i] = type_of(in[i]);
    }
    if (clip && to) {
        // of what is read where it lies; the copies made above are nobody else's, and of tensors that are not dense the bytes that they
        // count are not those that they reach over
        std::vector<Range> written = ranges_of(out);
        std::sort(written.begin(), written.end(), [](const Range &a, const Range &b) { return a.from < b.from; });
        for (size_t k = 1; k < written.size(); k++)
            if (written[k].from < written[k - 1].end) throw py::value_error("two tensors that clip_grad_norm writes share memory");
        for (const Range &r : ranges_of(in)) {
            // the written ones that end past r's begin: those from here on
            auto w = std::upper_bound(written.begin(), written.end(), r.from, [](uintptr_t p, const Range &b) { return p < b.end; });
            for (; w != written.end() && w->from < r.end; ++w)
                if (w->i != r.i || w->from != r.from) throw py::value_error("clip_grad_norm would write into memory of another of its tensors");
        }
    }
    Tensor norm = empty(first, {}, at::kFloat);
    const int64_t need = api.clip_scratch(sizes.data(), (int)sizes.size());
    const Tensor scratch = scratch_of(first, need);
    check(api.clip_grad_norm(from.data(), sizes.data(), types.data(), (int)sizes.size(), most, clip ? into.data() : nullptr,
                             norm.data_ptr<float>(), ptr(scratch), need, stream_of(first)));
    if (clip && to)
        for (const Tensor &t : out)
            if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
    return {out, norm};
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

bool vector_like(const Maybe &t, const Tensor &x, int64_t n) {
    return !t || ((like(*t, x, at::kFloat, 1) || like(*t, x, x.scalar_type(), 1)) && t->size(0) == n);
}
Maybe plain_layer_norm(const Tensor &x, const Maybe &w, const Maybe &b, double eps) {
    if (!floats(x, 2) || !within(x.size(1), 1, YGG_MOST_INNER) || !vector_like(w, x, x.size(1)) || !vector_like(b, x, x.size(1)) ||
        (w && b && w->scalar_type() != b->scalar_type()) || !(eps >= 0) || !(eps <= 1e30))
        return std::nullopt;
    return layer_norm(x, w, b, eps);
}
std::optional<std::pair<Tensor, Tensor>> plain_gated_scan(const Tensor &gate, const Tensor &x, const Maybe &state) {
    if (!floats(x, 3) || !(like(gate, x, at::kFloat, 3) || like(gate, x, x.scalar_type(), 3)) || gate.sizes() != x.sizes() ||
        !within(x.size(0), 0, YGG_MOST_ROWS) || !within(x.size(1), 0, YGG_MOST_STEPS) || !within(x.size(2), 1, YGG_MOST_INNER))
        return std::nullopt;
    if (state && !(like(*state, x, at::kFloat, 2) && state->size(0) == x.size(0) && state->size(1) == x.size(2))) return std::nullopt;
    return gated_scan(gate, x, state);
}
std::optional<std::pair<std::vector<Tensor>, Tensor>> plain_clip_grad_norm(const std::vector<Tensor> &in, double most, bool clip,
                                                                          const std::optional<std::vector<Tensor>> &to) {
    if (in.empty() || !(most >= 0) || (to && to->size() != in.size())) return std::nullopt;
    const bool grad = at::GradMode::is_enabled();
    auto plain = [&](const Tensor &t) {
        const auto d = t.scalar_type();
        return t.is_cuda() && t.layout() == at::kStrided && (d == at::kFloat || d == at::kBFloat16 || d == at::kHalf) &&
               t.device() == in[0].device() && t.numel() <= YGG_MOST_VALUES && !(clip && grad && t.requires_grad());
    };
    for (size_t i = 0; i < in.size(); i++) {
        if (!plain(in[i])) return std::nullopt;
        if (to && ((*to)[i].scalar_type() != in[i].scalar_type() || (*to)[i].sizes() != in[i].sizes() || !plain((*to)[i]))) return std::nullopt;
    }
    return clip_grad_norm(in, most, clip, to);
}
Maybe plain_gated_linear(const Tensor &x, const Tensor &w, int64_t act) {
    if (!floats(x, 2) || !like(w, x, x.scalar_type(), 3) || w.size(0) != 2 || w.size(2) != x.size(1) || x.size(0) > YGG_MOST_ROWS ||
        !within(w.size(1), 1, YGG_MOST_INNER / 2) || !within(x.size(1), 1, YGG_MOST_INNER))
        return std::nullopt;
    return gated_linear(x, w, act);
}

}  // namespace

PYBIND11_MODULE(_ygg_torch, m) {
    m.def("bind", &bind);
    m.def("token_logprobs", &token_logprobs);
    m.def("grouped_matmul", &grouped_matmul);
    m.def("int8_linear", &int8_linear);
    m.def("layer_norm", &layer_norm);
    m.def("gated_scan", &gated_scan);
    m.def("gated_linear", &gated_linear);
    m.def("clip_grad_norm", &clip_grad_norm);
    m.def("plain_token_logprobs", &plain_token_logprobs);
    m.def("plain_grouped_matmul", &plain_grouped_matmul);
    m.def("plain_int8_linear", &plain_int8_linear);
    m.def("plain_layer_norm", &plain_layer_norm);
    m.def("plain_gated_scan", &plain_gated_scan);
    m.def("plain_gated_linear", &plain_gated_linear);
    m.def("plain_clip_grad_norm", &plain_clip_grad_norm);
}
