// hip_policy.h — the policy's end of the VecEnv loop for C++ trainers: logits to actions, their scores with gradients, dropout, as torch::Tensor
// functions over the C ABI in include/gymhip.h (formulas there).  Header-only; gym_amd.policy (Python) binds these very functions.
//
// The reference leaves this to its trainer: VecEnv::step takes finished actions (wrappers/vec_env/base.h:56-63).  A step with a policy is
//     auto [actions, log_prob] = gym::policy::sampleActions(logits, {}, {.seed = 7, .row = env_offset, .step = t});
//     auto r = venv->step(actions);
// and its update scores the same actions again: actionLogProb(logits, actions) is differentiable in the logits.
//
// Everything runs on the logits' device and its current stream; nothing synchronises.  Wrong arguments throw std::invalid_argument, a call that
// fails or finds no GPU throws gym::policy::Error.
#pragma once
#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>
#include <torch/torch.h>

#include <cmath>
#include <limits>
#include <sstream>
#include <stdexcept>
#include <string>
#include <tuple>
#include <vector>

#include "gymhip.h"

namespace gym { namespace policy {

struct Error : std::runtime_error { using std::runtime_error::runtime_error; };

namespace detail {

[[noreturn]] inline void refuse(const std::string& what) { throw std::invalid_argument(what); }
inline void require(bool ok, const std::string& what) { if (!ok) refuse(what); }
inline void check(int rc, const char* what) {
    if (rc != GYMHIP_OK) throw Error(std::string(what) + " failed (code " + std::to_string(rc) + "): " + gymhip_last_error());
}

inline int typeOf(at::ScalarType t) { return t == at::kFloat ? GYMHIP_TYPE_F32 : t == at::kHalf ? GYMHIP_TYPE_F16 : t == at::kBFloat16 ? GYMHIP_TYPE_BF16 : -1; }

inline std::string shapeOf(at::IntArrayRef s) {
    std::string r = "(";
    for (size_t i = 0; i < s.size(); i++) r += (i ? ", " : "") + std::to_string(s[i]);
    return r + ")";
}

// x itself where its columns are adjacent and its rows lie in order (they may be apart, or all the same one); else a copy.
inline at::Tensor rowwise(const at::Tensor& x) {
    return (x.stride(1) == 1 || x.size(1) == 1) && x.stride(0) >= 0 ? x : x.contiguous();
}

// Forward-mode derivatives are not made, and what carries a tangent has no requires_grad to tell: refused, where its tangent would be lost.
inline void noTangent(const at::Tensor& x, const char* what) {
    if (x._fw_grad(0).defined()) throw std::runtime_error(std::string(what) + " carries a forward-mode derivative, which the policy operators do not have");
}

// derived: the result has a derivative in x.
inline at::Tensor ready(const at::Tensor& x, const char* what, bool derived = true) {
    if (x.dim() != 2) refuse(std::string(what) + " must be a 2-D tensor [rows, width]");
    if (typeOf(x.scalar_type()) < 0) refuse(std::string(what) + " must be float32, float16 or bfloat16, got " + at::toString(x.scalar_type()));
    if (derived) noTangent(x, what);
    if (!x.is_cuda()) throw Error(std::string(what) + " is on " + x.device().str() + ": the policy kernels run on the GPU and have no CPU fallback");
    if (x.size(1) > GYMHIP_POLICY_MAX_WIDTH) refuse(std::string(what) + ": at most 2^24 columns, got " + std::to_string(x.size(1)));
    return rowwise(x);
}

// A tensor beside the logits: its type, device and shape checked; adjacent along its last axis.  derived: the result has derivatives, but
// not in t, whose own would be lost.
inline at::Tensor side(const at::Tensor& t, const char* what, const at::Device& device, std::initializer_list<at::ScalarType> types,
                       std::initializer_list<std::vector<int64_t>> shapes, bool derived = true) {
    bool ok = false;
    std::string names;
    for (auto s : types) { ok = ok || t.scalar_type() == s; names += (names.empty() ? "" : " or ") + std::string(at::toString(s)); }
    require(ok, std::string(what) + " must be a tensor of " + names);
    require(t.device() == device, std::string(what) + " is on " + t.device().str() + ", the logits on " + device.str());
    if (derived) {
        require(!(t.requires_grad() && at::GradMode::is_enabled()), std::string(what) + " requires a gradient: only the logits have one");
        noTangent(t, what);
    }
    ok = false;
    names.clear();
    for (auto const& s : shapes) { ok = ok || t.sizes() == at::IntArrayRef(s); names += (names.empty() ? "" : " or ") + shapeOf(s); }
    require(ok, std::string(what) + " has shape " + shapeOf(t.sizes()) + ", expected " + names);
    return t.dim() == 0 || t.size(-1) <= 1 || t.stride(-1) == 1 ? t : t.contiguous();
}

inline int intType(const at::Tensor& t) { return t.scalar_type() == at::kLong ? GYMHIP_ACT_I64 : GYMHIP_ACT_I32; }
inline void* stream(const at::Tensor& x) { return (void*)c10::hip::getCurrentHIPStreamMasqueradingAsCUDA(x.device().index()).stream(); }
// t is written through its pointer, which autograd does not see: whoever has saved it (or a view of it) has to find it changed.  Inference tensors cannot be saved.
inline void written(const at::Tensor& t) { if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version(); }
inline at::Tensor emptyLike(const at::Tensor& x) { return at::empty(x.sizes(), x.options()); }

}  // namespace detail

// A number, or float32 [rows].
struct PerRow {
    double number = 0;
    at::Tensor rows;
    PerRow(double n) : number(n) {}
    PerRow(at::Tensor t) : rows(std::move(t)) {
        if (!rows.defined()) detail::refuse("a number per row is an undefined tensor");   // it would stand for the number 0: a greedy temperature
    }
};

// What is done to a row's logits before anything is chosen or scored: gymhip_logit_rules in tensors.
//   mask int32 [1 | rows | lines, words], mask_rows int32 [rows]; bias float32 [width], [1, width] or [rows, width];
//   history int32 / int64 [rows, length], history_len int32 / int64 [rows].  The tensors are read when an operator runs; their values are not checked.
struct LogitRules {
    at::Tensor mask, mask_rows, bias, history, history_len;
    PerRow repetition{1.0}, presence{0.0}, frequency{0.0}, temperature{1.0};

    void check() const {
        detail::require(mask.defined() || !mask_rows.defined(), "mask_rows without a mask");
        detail::require(history.defined() || !history_len.defined(), "history_len without a history");
        number(repetition, "repetition", true, false);
        number(presence, "presence", false, false);
        number(frequency, "frequency", false, false);
        number(temperature, "temperature", false, true);
    }
    std::vector<at::Tensor> tensors() const {
        std::vector<at::Tensor> all;
        for (auto const& t : {mask, mask_rows, bias, history, history_len, repetition.rows, presence.rows, frequency.rows, temperature.rows})
            if (t.defined()) all.push_back(t);
        return all;
    }

private:
    static void number(const PerRow& v, const char* name, bool positive, bool not_negative) {
        if (v.rows.defined()) return;
        // as the kernels take it: a number too small for float32 must not turn into the 0 that stands for something else
        const bool fits = std::abs(v.number) <= std::numeric_limits<float>::max(), positive_f = (float)v.number > 0;
        if (fits && (!positive || positive_f) && (!not_negative || positive_f || v.number == 0)) return;
        std::ostringstream what;
        what << name << " must be a finite float32" << (positive ? ", and positive" : not_negative ? ", and not negative" : "") << "; got " << v.number;
        detail::refuse(what.str());
    }
};

namespace detail {

// The rules for given logits as the C ABI takes them, and the tensors that this points into.
struct Bound : torch::CustomClassHolder {
    gymhip_logit_rules c{};
    bool any = false;
    std::vector<at::Tensor> keep;
    const gymhip_logit_rules* ptr() const { return any ? &c : nullptr; }

    Bound() = default;
    Bound(const LogitRules& r, const at::Tensor& logits, bool derived = true) : any(true) {
        r.check();
        const int64_t rows = logits.size(0), width = logits.size(1), words = (width + 31) / 32;
        const at::Device dev = logits.device();
        c.struct_size = (int32_t)sizeof c;
        if (r.mask.defined()) {
            require(r.mask.dim() == 2 && r.mask.size(1) >= words, "mask must be an int32 tensor [lines, >= " + std::to_string(words) + "] for " + std::to_string(width) + " columns");
            require(r.mask_rows.defined() || r.mask.size(0) == 1 || r.mask.size(0) == rows,
                    "mask has " + std::to_string(r.mask.size(0)) + " lines for " + std::to_string(rows) + " rows: one, one per row, or mask_rows");
            require(r.mask.size(0) > 0 || rows == 0, "mask has no lines");
            at::Tensor m = side(r.mask, "mask", dev, {at::kInt}, {r.mask.sizes().vec()});
            if (m.size(0) > 1 && m.stride(0) < words) m = m.contiguous();   // lines that share storage (an expanded mask)
            c.mask = (const uint32_t*)held(m);
            c.mask_stride = m.stride(0);
            c.mask_lines = m.size(0);
            if (r.mask_rows.defined()) c.mask_rows = (const int32_t*)held(side(r.mask_rows, "mask_rows", dev, {at::kInt}, {{rows}}));
        }
        if (r.bias.defined()) {
            at::Tensor b = side(r.bias, "bias", dev, {at::kFloat}, {{width}, {1, width}, {rows, width}}, derived);
            if (b.dim() == 2 && b.stride(0) < 0) b = b.contiguous();
            c.bias = (const float*)held(b);
            c.bias_stride = b.dim() == 2 && b.size(0) > 1 ? b.stride(0) : 0;
        }
        if (r.history.defined()) {
            require(r.history.dim() == 2 && r.history.size(0) == rows, "history must be an int32 or int64 tensor [" + std::to_string(rows) + ", length]");
            const at::Tensor h = side(r.history, "history", dev, {at::kInt, at::kLong}, {r.history.sizes().vec()});
            if (h.size(1) > 0) {
                c.history = held(h);
                c.history_dtype = intType(h);
                c.history_stride = h.stride(0);
                c.history_cols = h.size(1);
            }
            if (r.history_len.defined()) {
                const at::Tensor n = side(r.history_len, "history_len", dev, {at::kInt, at::kLong}, {{rows}});
                if (c.history) {
                    c.history_len = held(n);
                    c.history_len_dtype = intType(n);
                }
            }
        }
        value(r.repetition, "repetition", rows, dev, derived, &c.repetition, &c.repetition_rows);
        value(r.presence, "presence", rows, dev, derived, &c.presence, &c.presence_rows);
        value(r.frequency, "frequency", rows, dev, derived, &c.frequency, &c.frequency_rows);
        value(r.temperature, "temperature", rows, dev, derived, &c.temperature, &c.temperature_rows);
        any = rows > 0 && width > 0;   // of an empty batch the tensors are checked and no more: their pointers are null, which stands for no rule
    }

private:
    const void* held(const at::Tensor& t) {
        keep.push_back(t);
        return t.data_ptr();
    }
    void value(const PerRow& v, const char* name, int64_t rows, const at::Device& dev, bool derived, float* number, const float** per_row) {
        if (v.rows.defined()) *per_row = (const float*)held(side(v.rows, name, dev, {at::kFloat}, {{rows}}, derived));
        else *number = (float)v.number;
    }
};
using BoundPtr = c10::intrusive_ptr<Bound>;
inline BoundPtr bind(const LogitRules* rules, const at::Tensor& logits, bool derived = true) {
    return rules ? c10::make_intrusive<Bound>(*rules, logits, derived) : c10::make_intrusive<Bound>();
}

}  // namespace detail

// Which random numbers a row draws: a function of (seed, row key, step) alone.  `rows` int64 [rows] in place of row, row + 1, ..; `steps` int64, one
// (read when the kernel runs: advance it between replays of a recorded graph) or [rows], in place of `step`.
struct Keys {
    uint64_t seed = 0;
    int64_t row = 0, step = 0;
    at::Tensor rows, steps;
};

namespace detail {
struct BoundKeys : torch::CustomClassHolder {
    gymhip_random_keys c{};
    std::vector<at::Tensor> keep;
    BoundKeys(const Keys& k, int64_t n, const at::Device& dev) {
        c.struct_size = (int32_t)sizeof c;
        c.seed = k.seed;
        c.row = k.row;
        c.step = k.step;
        if (k.rows.defined()) {
            keep.push_back(side(k.rows, "rows", dev, {at::kLong}, {{n}}));
            c.rows = keep.back().data_ptr<int64_t>();
        }
        if (k.steps.defined()) {
            keep.push_back(side(k.steps, "step", dev, {at::kLong}, {{}, {1}, {n}}));
            c.steps = keep.back().data_ptr<int64_t>();
            c.steps_per_row = k.steps.dim() == 1 && k.steps.size(0) == n;
        }
    }
};

inline void once() {
    if (at::GradMode::is_enabled()) throw std::runtime_error("the policy operators are differentiable once: create_graph is not available");
}
inline bool graded(const at::Tensor& x) { return x.requires_grad() && at::GradMode::is_enabled(); }

inline void process(const at::Tensor& x, const Bound& b, at::Tensor& out) {
    const c10::OptionalDeviceGuard guard(x.device());
    check(gymhip_process_logits(x.data_ptr(), typeOf(x.scalar_type()), x.size(0), x.size(1), x.stride(0), b.ptr(), out.data_ptr(), out.stride(0), stream(x)),
          "gymhip_process_logits");
}

struct ProcessFunction : torch::autograd::Function<ProcessFunction> {
    static at::Tensor forward(torch::autograd::AutogradContext* ctx, const at::Tensor& logits, const BoundPtr& b, const std::vector<at::Tensor>& tensors) {
        const at::Tensor x = rowwise(logits);
        at::Tensor out = emptyLike(x);
        process(x, *b, out);
        // the rules' tensors are saved too, so that changing one in place before the backward pass is an error
        torch::autograd::variable_list saved{x};
        saved.insert(saved.end(), tensors.begin(), tensors.end());
        ctx->save_for_backward(std::move(saved));
        ctx->saved_data["rules"] = c10::IValue::make_capsule(b);
        return out;
    }
    static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, torch::autograd::variable_list grads) {
        once();
        const auto saved = ctx->get_saved_variables();
        const auto b = c10::static_intrusive_pointer_cast<Bound>(ctx->saved_data["rules"].toCapsule());
        const at::Tensor x = rowwise(saved[0]), g = rowwise(grads[0]);
        at::Tensor out = emptyLike(x);
        const c10::OptionalDeviceGuard guard(x.device());
        check(gymhip_process_logits_backward(x.data_ptr(), typeOf(x.scalar_type()), x.size(0), x.size(1), x.stride(0), b->ptr(), g.data_ptr(), g.stride(0),
                                             out.data_ptr(), out.stride(0), stream(x)), "gymhip_process_logits_backward");
        return {out, at::Tensor(), at::Tensor()};
    }
};

struct Scores { at::Tensor log_prob, entropy, log_sum; };
inline Scores score(const at::Tensor& x, const Bound& b, const at::Tensor& actions) {
    const int64_t n = x.size(0), width = x.size(1);
    const auto f = x.options().dtype(at::kFloat);
    Scores s{at::empty({n}, f), at::empty({n}, f), at::empty({n, 2}, x.options().dtype(at::kDouble))};
    const size_t bytes = gymhip_action_log_prob_workspace_bytes(n, width);
    const at::Tensor ws = bytes ? at::empty({(int64_t)bytes}, x.options().dtype(at::kByte)) : at::Tensor();
    const c10::OptionalDeviceGuard guard(x.device());
    check(gymhip_action_log_prob(x.data_ptr(), typeOf(x.scalar_type()), n, width, x.stride(0), b.ptr(), actions.data_ptr(), intType(actions),
                                 s.log_prob.data_ptr<float>(), s.entropy.data_ptr<float>(), s.log_sum.data_ptr<double>(), bytes ? ws.data_ptr() : nullptr,
                                 bytes, stream(x)), "gymhip_action_log_prob");
    return s;
}

struct ScoreFunction : torch::autograd::Function<ScoreFunction> {
    static torch::autograd::variable_list forward(torch::autograd::AutogradContext* ctx, const at::Tensor& logits, const at::Tensor& actions, const BoundPtr& b,
                                                  const std::vector<at::Tensor>& tensors) {
        ctx->set_materialize_grads(false);
        const at::Tensor x = rowwise(logits);
        const Scores s = score(x, *b, actions);
        torch::autograd::variable_list saved{x, actions, s.log_prob, s.entropy, s.log_sum};
        saved.insert(saved.end(), tensors.begin(), tensors.end());
        ctx->save_for_backward(std::move(saved));
        ctx->saved_data["rules"] = c10::IValue::make_capsule(b);
        return {s.log_prob, s.entropy};
    }
    static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, torch::autograd::variable_list grads) {
        once();
        const auto saved = ctx->get_saved_variables();
        const auto b = c10::static_intrusive_pointer_cast<Bound>(ctx->saved_data["rules"].toCapsule());
        const at::Tensor x = rowwise(saved[0]);
        at::Tensor out = emptyLike(x), g[2];
        for (int i = 0; i < 2; i++)
            if (grads[i].defined()) g[i] = grads[i].contiguous();
        const c10::OptionalDeviceGuard guard(x.device());
        check(gymhip_action_log_prob_backward(x.data_ptr(), typeOf(x.scalar_type()), x.size(0), x.size(1), x.stride(0), b->ptr(), saved[1].data_ptr(),
                                              intType(saved[1]), saved[2].data_ptr<float>(), saved[3].data_ptr<float>(), saved[4].data_ptr<double>(),
                                              g[0].defined() ? g[0].data_ptr<float>() : nullptr, g[1].defined() ? g[1].data_ptr<float>() : nullptr,
                                              out.data_ptr(), out.stride(0), stream(x)), "gymhip_action_log_prob_backward");
        return {out, at::Tensor(), at::Tensor(), at::Tensor()};
    }
};

inline at::Tensor drop(const at::Tensor& x, double p, const BoundKeys& k) {
    at::Tensor out = emptyLike(x);
    const c10::OptionalDeviceGuard guard(x.device());
    check(gymhip_dropout(x.data_ptr(), typeOf(x.scalar_type()), x.size(0), x.size(1), x.stride(0), p, &k.c, out.data_ptr(), out.stride(0), stream(x)),
          "gymhip_dropout");
    return out;
}

struct DropoutFunction : torch::autograd::Function<DropoutFunction> {
    static at::Tensor forward(torch::autograd::AutogradContext* ctx, const at::Tensor& x, double p, const c10::intrusive_ptr<BoundKeys>& k) {
        ctx->saved_data["p"] = p;
        ctx->saved_data["keys"] = c10::IValue::make_capsule(k);   // holds the tensors it points into
        ctx->save_for_backward(torch::autograd::variable_list(k->keep.begin(), k->keep.end()));   // a change in place before the backward pass is an error
        return drop(rowwise(x), p, *k);
    }
    static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, torch::autograd::variable_list grads) {
        once();
        ctx->get_saved_variables();
        const auto k = c10::static_intrusive_pointer_cast<BoundKeys>(ctx->saved_data["keys"].toCapsule());
        return {drop(rowwise(grads[0]), ctx->saved_data["p"].toDouble(), *k), at::Tensor(), at::Tensor()};
    }
};
}  // namespace detail

// z of the logits, rounded to float32 and from there to their type.  Differentiable in the logits.
inline at::Tensor processLogits(const at::Tensor& logits, const LogitRules* rules = nullptr) {
    const at::Tensor x = detail::ready(logits, "logits");
    const detail::BoundPtr b = detail::bind(rules, x);
    if (detail::graded(logits)) return detail::ProcessFunction::apply(logits, b, rules ? rules->tensors() : std::vector<at::Tensor>());
    at::Tensor out = detail::emptyLike(x);
    detail::process(x, *b, out);
    return out;
}
// The same into `out`, which may be the logits themselves, or memory that shares no element with them or the rules' tensors (other columns of the same buffer, say); not under autograd.  A change of `out` in place, for
// whoever has saved it for a backward pass.
inline void processLogitsInto(const at::Tensor& logits, const LogitRules* rules, at::Tensor out) {
    detail::noTangent(out, "out");
    const at::Tensor x = detail::ready(logits, "logits");
    detail::require(!at::GradMode::is_enabled() || !(logits.requires_grad() || out.requires_grad()), "out= is not available under autograd");
    detail::require(out.sizes() == logits.sizes() && out.scalar_type() == logits.scalar_type() && out.device() == logits.device() &&
                    (out.stride(1) == 1 || out.size(1) <= 1), "out must have the logits' shape, type and device, and adjacent columns");
    const detail::BoundPtr b = detail::bind(rules, x);
    detail::written(out);
    detail::process(x, *b, out);
}

// One action per row from softmax(z) (int32; -1 where nothing can be chosen) and its log-probability (float32, no gradient).  Into `actions` and `log_prob`
// where both are given, which is a change of them in place.
inline std::tuple<at::Tensor, at::Tensor> sampleActions(const at::Tensor& logits, const LogitRules* rules, const Keys& keys, at::Tensor actions = {},
                                                        at::Tensor log_prob = {}) {
    if (actions.defined() != log_prob.defined()) detail::refuse("out needs both actions and log_prob, or neither");
    const bool given = actions.defined();
    const at::Tensor x = detail::ready(logits, "logits", false);
    const int64_t n = x.size(0), width = x.size(1);
    if (given) {
        detail::side(actions, "out.actions", x.device(), {at::kInt}, {{n}});
        detail::side(log_prob, "out.log_prob", x.device(), {at::kFloat}, {{n}});
        detail::require(actions.is_contiguous() && log_prob.is_contiguous(), "out tensors must be contiguous");
    } else {
        actions = at::empty({n}, x.options().dtype(at::kInt));
        log_prob = at::empty({n}, x.options().dtype(at::kFloat));
    }
    const detail::BoundPtr b = detail::bind(rules, x, false);
    const detail::BoundKeys k(keys, n, x.device());
    const size_t bytes = gymhip_sample_workspace_bytes(n, width);
    const at::Tensor ws = bytes ? at::empty({(int64_t)bytes}, x.options().dtype(at::kByte)) : at::Tensor();
    if (given) {
        detail::written(actions);
        detail::written(log_prob);
    }
    const c10::OptionalDeviceGuard guard(x.device());
    detail::check(gymhip_sample_actions(x.data_ptr(), detail::typeOf(x.scalar_type()), n, width, x.stride(0), b->ptr(), &k.c, actions.data_ptr<int32_t>(),
                                        log_prob.data_ptr<float>(), bytes ? ws.data_ptr() : nullptr, bytes, detail::stream(x)), "gymhip_sample_actions");
    return {actions, log_prob};
}

// (log softmax(z)[action], entropy of softmax(z)), float32 [rows] each, for actions int32 / int64 [rows].  Differentiable in the logits.
inline std::tuple<at::Tensor, at::Tensor> actionLogProb(const at::Tensor& logits, const at::Tensor& actions_, const LogitRules* rules = nullptr) {
    const at::Tensor x = detail::ready(logits, "logits");
    const at::Tensor actions = detail::side(actions_, "actions", x.device(), {at::kInt, at::kLong}, {{x.size(0)}});
    const detail::BoundPtr b = detail::bind(rules, x);
    if (detail::graded(logits)) {
        auto r = detail::ScoreFunction::apply(logits, actions, b, rules ? rules->tensors() : std::vector<at::Tensor>());
        return {r[0], r[1]};
    }
    const detail::Scores s = detail::score(x, *b, actions);
    return {s.log_prob, s.entropy};
}

// x [rows, width] with each element 0 with probability p (to 16 bits), else multiplied by 65536 / (65536 - round(65536 p)).  Differentiable in x.
inline at::Tensor dropout(const at::Tensor& x_, double p, const Keys& keys) {
    const at::Tensor x = detail::ready(x_, "x");
    if (!(p >= 0 && p < 1 && std::nearbyint(65536 * p) <= 65535)) detail::refuse("p must lie in [0, 1) and round to less than 65536 / 65536, got " + std::to_string(p));
    auto k = c10::make_intrusive<detail::BoundKeys>(keys, x.size(0), x.device());
    return detail::graded(x_) ? detail::DropoutFunction::apply(x_, p, k) : detail::drop(x, p, *k);
}

}}  // namespace gym::policy
