// policy_torch.cpp — gym_amd.policy's binding of gym/hip_policy.h.  The autograd nodes are C++: an update of a small policy is bound by the host, and a
// Python node's backward pass alone costs as much as the rest of the call.
#include <torch/extension.h>

#include "gym/hip_policy.h"

namespace py = pybind11;
using namespace gym::policy;
// Tensors first: a tensor of one element would pass for a number (and be waited for).
using Number = std::variant<at::Tensor, double>;
using Index = std::variant<at::Tensor, int64_t>;

static PerRow perRow(const Number& v) { return std::holds_alternative<double>(v) ? PerRow(std::get<double>(v)) : PerRow(std::get<at::Tensor>(v)); }
static py::object numberOf(const PerRow& v) { return v.rows.defined() ? py::cast(v.rows) : py::cast(v.number); }
static at::Tensor given(const std::optional<at::Tensor>& t) { return t ? *t : at::Tensor(); }

static Keys keys(const py::int_& seed, const Index& step, const Index& rows) {
    Keys k;
    k.seed = PyLong_AsUnsignedLongLongMask(seed.ptr());
    if (PyErr_Occurred()) throw py::error_already_set();
    if (std::holds_alternative<int64_t>(step)) k.step = std::get<int64_t>(step);
    else k.steps = std::get<at::Tensor>(step);
    if (std::holds_alternative<int64_t>(rows)) k.row = std::get<int64_t>(rows);
    else k.rows = std::get<at::Tensor>(rows);
    return k;
}

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
    py::register_exception_translator([](std::exception_ptr p) {
        try {
            if (p) std::rethrow_exception(p);
        } catch (const Error& e) {
            py::set_error(py::module_::import("gym_amd._lib").attr("GymhipError"), e.what());
        }
    });
    py::class_<LogitRules> rules(m, "LogitRules");
    rules.def(py::init([](const std::optional<at::Tensor>& mask, const std::optional<at::Tensor>& mask_rows, const std::optional<at::Tensor>& bias,
                          const std::optional<at::Tensor>& history, const std::optional<at::Tensor>& history_len, const Number& repetition, const Number& presence,
                          const Number& frequency, const Number& temperature) {
                  LogitRules r{given(mask), given(mask_rows), given(bias), given(history), given(history_len), perRow(repetition), perRow(presence),
                               perRow(frequency), perRow(temperature)};
                  r.check();
                  return r;
              }),
              py::kw_only(), py::arg("mask") = py::none(), py::arg("mask_rows") = py::none(), py::arg("bias") = py::none(), py::arg("history") = py::none(),
              py::arg("history_len") = py::none(), py::arg("repetition") = 1.0, py::arg("presence") = 0.0, py::arg("frequency") = 0.0,
              py::arg("temperature") = 1.0);
#define FIELD(name)                                                                                                              \
    rules.def_property(#name, [](const LogitRules& r) { return r.name.defined() ? py::cast(r.name) : py::object(py::none()); }, \
                       [](LogitRules& r, const std::optional<at::Tensor>& t) { r.name = given(t); })
    FIELD(mask); FIELD(mask_rows); FIELD(bias); FIELD(history); FIELD(history_len);
#undef FIELD
#define FIELD(name) \
    rules.def_property(#name, [](const LogitRules& r) { return numberOf(r.name); }, [](LogitRules& r, const Number& v) { r.name = perRow(v); })
    FIELD(repetition); FIELD(presence); FIELD(frequency); FIELD(temperature);
#undef FIELD
    // The checks alone, and what the kernels would be handed (tests of the host side).
    rules.def("_bind", [](const LogitRules& r, const at::Tensor& logits) {
        const gym::policy::detail::Bound b(r, logits);
        using namespace py::literals;
        py::object c = py::module_::import("types").attr("SimpleNamespace")("mask_stride"_a = b.c.mask_stride, "mask_lines"_a = b.c.mask_lines,
            "bias_stride"_a = b.c.bias_stride, "history"_a = b.c.history != nullptr, "history_stride"_a = b.c.history_stride, "history_cols"_a = b.c.history_cols);
        return py::make_tuple(c, b.keep);
    });
    m.def("process_logits", &processLogits, py::arg("logits"), py::arg("rules").none(true));
    m.def("process_logits_into", &processLogitsInto, py::arg("logits"), py::arg("rules").none(true), py::arg("out"));
    m.def("sample_actions", [](const at::Tensor& logits, const LogitRules* r, const py::int_& seed, const Index& step, const Index& rows,
                               const std::optional<at::Tensor>& actions, const std::optional<at::Tensor>& log_prob) {
        return sampleActions(logits, r, keys(seed, step, rows), given(actions), given(log_prob));
    }, py::arg("logits"), py::arg("rules").none(true), py::arg("seed"), py::arg("step"), py::arg("rows"), py::arg("actions") = py::none(),
       py::arg("log_prob") = py::none());
    m.def("action_log_prob", &actionLogProb, py::arg("logits"), py::arg("actions"), py::arg("rules").none(true));
    m.def("dropout", [](const at::Tensor& x, double p, const py::int_& seed, const Index& step, const Index& rows) { return dropout(x, p, keys(seed, step, rows)); });
}
