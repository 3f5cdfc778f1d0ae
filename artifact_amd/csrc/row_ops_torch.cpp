// The row operators of include/rof.h as differentiable PyTorch functions: the compiled half of artifact_amd/row_ops.py.
// They are written in C++ because small graphs are a matter of the host: a step of 16384 x 16 floats is 15 us on the device,
// and as Python functions the operators' forward and backward calls alone took 147 us of the host's time (here 60, most of it
// the autograd engine's).
//
// Nothing but the inputs is kept for the backward pass.  Checks raise the exception type that set_error_type was given.
//
// They are registered with PyTorch's dispatcher (rof::layer_norm, rof::layer_norm_backward, rof::dropout,
// rof::dropout_state_next), and every call goes through it, the backward pass's too.  What records a program from the calls
// it sees (torch.jit.trace, make_fx) then sees these; without them it would see no more than the allocation of the
// result, and replay that.  A replay calls the operators with other tensors, so the checks are theirs.
//
// Built by artifact_amd/build.py into artifact_amd/_ROFrows*.so.
#include <torch/extension.h>
#include <torch/library.h>

#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/graph_task.h>
#include <torch/csrc/autograd/saved_variable.h>

#include <cmath>
#include <memory>
#include <mutex>
#include <optional>
#include <stdexcept>
#include <string>

#include "rof.h"

namespace {

using at::Tensor;
using torch::autograd::Node;
using torch::autograd::SavedVariable;
using torch::autograd::variable_list;

PyObject *g_error_type = nullptr;

struct Failure : std::runtime_error {
    using std::runtime_error::runtime_error;
};

void require(bool ok, const char *message) {
    if (!ok) throw Failure(message);
}
void require(bool ok, const char *name, const char *message) {
    if (!ok) throw Failure(std::string(name) + message);
}

void check(int rc, const char *what) {
    if (rc == ROF_OK) return;
    std::string msg = std::string("librof: ") + what + ": " + rof_strerror(rc);
    if (rc == ROF_ERR_DEVICE) msg += std::string(": ") + rof_last_device_error();
    throw Failure(msg + " (status " + std::to_string(rc) + ")");
}

void *current_stream(const Tensor &t) { return (void *)c10::hip::getCurrentHIPStream(t.get_device()).stream(); }

int type_of(at::ScalarType t) { return t == at::kFloat ? ROF_F32 : ROF_BF16; }
bool known(at::ScalarType t) { return t == at::kFloat || t == at::kBFloat16; }
int64_t row_stride(const Tensor &t) { return t.size(0) > 1 ? t.stride(0) : std::max(t.stride(0), t.size(1)); }
bool rows_apart(const Tensor &t) {
    return (t.size(1) <= 1 || t.stride(1) == 1) && (t.size(0) <= 1 || t.stride(0) >= t.size(1));
}
void *address(const Tensor &t) { return t.defined() ? t.data_ptr() : nullptr; }

void check_tangent(const char *name, const Tensor &t) {
    require(!t._fw_grad(0).defined(), name, " must not carry a forward-mode tangent (there is no forward-mode derivative)");
}
void check_rows(const char *name, const Tensor &t) {
    require(t.is_cuda() && t.dim() == 2 && known(t.scalar_type()), name, " must be a 2-D float32 or bfloat16 CUDA tensor");
    require(t.size(1) > 0 && t.size(1) <= INT32_MAX, name, " must have at least one column");
    require(rows_apart(t), name, " must have unit column stride and rows that do not overlap");
    require(!t.is_neg(), name, " must not be a view with the negative bit (resolve it first)");
    check_tangent(name, t);
}
void check_param(const char *name, const Tensor &t, const Tensor &x) {
    require(!t.defined() || (t.scalar_type() == at::kFloat && t.device() == x.device() && t.dim() == 1 &&
                             t.numel() == x.size(1) && t.is_contiguous() && !t.is_neg()),
            name, " must be a contiguous float32 vector with one element per column on the device of x");
    if (t.defined()) check_tangent(name, t);
}
void check_rate(double p) { require(p >= 0.0 && p <= 1.0, "a dropout rate must lie between 0 and 1"); }
void check_rng(const Tensor &rng, const Tensor &x) {
    require(rng.defined(), "dropout needs rng: an int64 tensor {seed, offset} on the device of x (see ROF_DropoutState)");
    require(rng.scalar_type() == at::kLong && rng.device() == x.device() && rng.numel() == 2 && rng.is_contiguous() &&
                !rng.is_neg(),
            "rng must be a contiguous int64 tensor of two elements {seed, offset} on the device of x");
}

// An incoming gradient as rows the kernels take: autograd hands over broadcast and transposed ones as well.
Tensor gradient_rows(Tensor grad, at::ScalarType type) {
    check_tangent("the gradient", grad);
    grad = grad.resolve_neg();
    if (grad.scalar_type() != type) grad = grad.to(type);
    return rows_apart(grad) ? grad : grad.contiguous();
}

// Gradients of a pass that is itself recorded (create_graph): differentiating them is an error, not a silent zero.
variable_list once(variable_list grads, const char *what) {
    if (!at::GradMode::is_enabled()) return grads;
    for (auto &g : grads)
        if (g.defined()) {
            auto fail = std::make_shared<torch::autograd::DelayedError>(std::string(what) + " has no second derivative", 1);
            g = g.detach();
            g.set_requires_grad(true);
            g = (*fail)({g})[0];
        }
    return grads;
}

using LayerNorm = Tensor(const Tensor &, const std::optional<Tensor> &, const std::optional<Tensor> &, double, bool, double,
                         const std::optional<Tensor> &, int64_t, std::optional<at::ScalarType>);
using LayerNormBackward = std::tuple<Tensor, Tensor, Tensor>(const Tensor &, const Tensor &, const std::optional<Tensor> &,
                                                             const std::optional<Tensor> &, double, bool, double,
                                                             const std::optional<Tensor> &, int64_t, at::ScalarType, bool, bool,
                                                             bool);
using Dropout = Tensor(const Tensor &, double, const std::optional<Tensor> &, int64_t);
using DropoutStateNext = Tensor(const Tensor &, int64_t);

template <typename F>
c10::TypedOperatorHandle<F> find(const char *name) {
    return c10::Dispatcher::singleton().findSchemaOrThrow(name, "").typed<F>();
}
const auto &layer_norm_op() {
    static const auto op = find<LayerNorm>("rof::layer_norm");
    return op;
}
const auto &layer_norm_backward_op() {
    static const auto op = find<LayerNormBackward>("rof::layer_norm_backward");
    return op;
}
const auto &dropout_op() {
    static const auto op = find<Dropout>("rof::dropout");
    return op;
}
const auto &dropout_state_next_op() {
    static const auto op = find<DropoutStateNext>("rof::dropout_state_next");
    return op;
}

std::optional<Tensor> maybe(const Tensor &t) { return t.defined() ? std::optional<Tensor>(t) : std::nullopt; }

// What the checks of the kernels below would not be reached with, or too late to be told plainly.
void check_call(const Tensor &x) {
    require(x.is_cuda() && x.layout() == at::kStrided, "x must be a 2-D float32 or bfloat16 CUDA tensor");
}
void check_plain(const std::optional<Tensor> &t) {
    const c10::DispatchKeySet wrapped({c10::DispatchKey::FuncTorchBatched, c10::DispatchKey::FuncTorchGradWrapper});
    require(!t || !t->key_set().has_any(wrapped), "the row operators do not take part in torch.func's transforms");
}

// ---- on the device ------------------------------------------------------------------------------------------------
Tensor dropout_cuda(const Tensor &x, double p, const std::optional<Tensor> &rng_, int64_t call) {
    const Tensor rng = rng_.value_or(Tensor());
    check_rows("x", x);
    check_rate(p);
    check_rng(rng, x);
    const c10::DeviceGuard guard(x.device());
    Tensor out = at::empty({x.size(0), x.size(1)}, x.options());
    const rof_dropout_opts opts = {p, (const int64_t *)rng.data_ptr(), call};
    check(rof_dropout(x.data_ptr(), type_of(x.scalar_type()), row_stride(x), x.size(0), (int)x.size(1), out.data_ptr(), x.size(1),
                      &opts, current_stream(x)),
          "dropout");
    return out;
}

void check_norm(const Tensor &x, const Tensor &weight, const Tensor &bias, double eps, double p, const Tensor &rng,
                at::ScalarType out_type) {
    check_rows("x", x);
    require(x.size(1) * (int64_t)x.element_size() <= ROF_LAYER_NORM_MAX_ROW_BYTES,
            "layer_norm takes rows of at most 32768 bytes (8192 float32 or 16384 bfloat16 columns)");
    static_assert(ROF_LAYER_NORM_MAX_ROW_BYTES == 32768, "the message above");
    check_param("weight", weight, x);
    check_param("bias", bias, x);
    require(eps >= 0.0 && eps <= 1e30, "eps must not be negative, and finite");
    check_rate(p);
    if (p > 0) check_rng(rng, x);
    require(known(out_type), "out_dtype must be float32 or bfloat16");
}

Tensor layer_norm_cuda(const Tensor &x, const std::optional<Tensor> &weight_, const std::optional<Tensor> &bias_, double eps,
                       bool relu, double p, const std::optional<Tensor> &rng_, int64_t call,
                       std::optional<at::ScalarType> out_type_) {
    const Tensor weight = weight_.value_or(Tensor()), bias = bias_.value_or(Tensor()), rng = rng_.value_or(Tensor());
    const at::ScalarType out_type = out_type_.value_or(x.scalar_type());
    check_norm(x, weight, bias, eps, p, rng, out_type);
    const c10::DeviceGuard guard(x.device());
    Tensor out = at::empty({x.size(0), x.size(1)}, x.options().dtype(out_type));
    const rof_dropout_opts opts = {p, p > 0 ? (const int64_t *)rng.data_ptr() : nullptr, call};
    check(rof_layer_norm(x.data_ptr(), type_of(x.scalar_type()), row_stride(x), x.size(0), (int)x.size(1),
                         (const float *)address(weight), (const float *)address(bias), eps, relu, p > 0 ? &opts : nullptr,
                         out.data_ptr(), type_of(out_type), x.size(1), current_stream(x)),
          "layer norm");
    return out;
}

// out_type: that of the forward pass's result, which the gradient is taken to
std::tuple<Tensor, Tensor, Tensor> layer_norm_backward_cuda(const Tensor &grad_, const Tensor &x, const std::optional<Tensor> &weight_,
                                                            const std::optional<Tensor> &bias_, double eps, bool relu, double p,
                                                            const std::optional<Tensor> &rng_, int64_t call,
                                                            at::ScalarType out_type, bool want_x, bool want_weight, bool want_bias) {
    const Tensor weight = weight_.value_or(Tensor()), bias = bias_.value_or(Tensor()), rng = rng_.value_or(Tensor());
    check_norm(x, weight, bias, eps, p, rng, out_type);
    require(grad_.device() == x.device() && grad_.sizes() == x.sizes(), "the gradient must be of x's shape and on its device");
    const c10::DeviceGuard guard(x.device());
    const Tensor grad = gradient_rows(grad_, out_type);
    const int64_t n = x.size(0), f = x.size(1);
    const auto floats = x.options().dtype(at::kFloat);
    Tensor dx, dw, db, workspace;
    if (want_x) dx = at::empty({n, f}, x.options());
    if (want_weight) dw = at::empty({f}, floats);
    if (want_bias) db = at::empty({f}, floats);
    const size_t bytes = want_weight || want_bias ? rof_layer_norm_backward_workspace_bytes(n, (int)f) : 0;
    if (bytes) workspace = at::empty({(int64_t)(bytes / sizeof(float))}, floats);
    const rof_dropout_opts opts = {p, p > 0 ? (const int64_t *)rng.data_ptr() : nullptr, call};
    check(rof_layer_norm_backward(grad.data_ptr(), type_of(out_type), row_stride(grad), x.data_ptr(), type_of(x.scalar_type()),
                                  row_stride(x), n, (int)f, (const float *)address(weight), (const float *)address(bias), eps, relu,
                                  p > 0 ? &opts : nullptr, address(dx), f, (float *)address(dw), (float *)address(db),
                                  address(workspace), bytes, current_stream(x)),
          "layer norm's gradient");
    return {dx, dw, db};
}

// ---- differentiation ----------------------------------------------------------------------------------------------
struct RofDropoutBackward : public Node {
    SavedVariable rng;
    double p;
    int64_t call;
    at::ScalarType type;

    variable_list apply(variable_list &&grads) override {
        std::lock_guard<std::mutex> lock(mutex_);
        if (!grads[0].defined()) return variable_list(1);
        const Tensor state = rng.unpack();   // outside the guards: a checkpointed part runs its forward pass again here
        Tensor dx;
        {
            at::NoGradGuard quiet;
            const Tensor rows = gradient_rows(grads[0], type);
            const at::AutoDispatchBelowADInplaceOrView below;
            dx = dropout_op().call(rows, p, maybe(state), call);
        }
        return once({dx}, "dropout");
    }
    void release_variables() override {
        std::lock_guard<std::mutex> lock(mutex_);
        rng.reset_data();
    }
    std::string name() const override { return "RofDropoutBackward"; }
};

Tensor dropout_autograd(const Tensor &x, double p, const std::optional<Tensor> &rng, int64_t call) {
    Tensor out;
    {
        const at::AutoDispatchBelowADInplaceOrView below;
        out = dropout_op().call(x, p, rng, call);
    }
    if (at::GradMode::is_enabled() && x.requires_grad()) {
        auto node = std::shared_ptr<RofDropoutBackward>(new RofDropoutBackward(), torch::autograd::deleteNode);
        node->set_next_edges(torch::autograd::collect_next_edges(x));
        node->rng = SavedVariable(rng.value_or(Tensor()), false);
        node->p = p;
        node->call = call;
        node->type = x.scalar_type();
        torch::autograd::set_history(out, node);
    }
    return out;
}

struct RofLayerNormBackward : public Node {
    SavedVariable x_, weight_, bias_, rng_;
    double eps, p;
    bool relu;
    int64_t call;
    at::ScalarType out_type;

    variable_list apply(variable_list &&grads) override {
        std::lock_guard<std::mutex> lock(mutex_);
        if (!grads[0].defined()) return variable_list(3);
        // outside the guards, as above
        const Tensor x = x_.unpack(), weight = weight_.unpack(), bias = bias_.unpack(), rng = rng_.unpack();
        std::tuple<Tensor, Tensor, Tensor> d;
        {
            at::NoGradGuard quiet;
            const at::AutoDispatchBelowADInplaceOrView below;
            d = layer_norm_backward_op().call(grads[0], x, maybe(weight), maybe(bias), eps, relu, p, maybe(rng), call, out_type,
                                              task_should_compute_output(0), task_should_compute_output(1),
                                              task_should_compute_output(2));
        }
        return once({std::get<0>(d), std::get<1>(d), std::get<2>(d)}, "layer_norm");
    }
    void release_variables() override {
        std::lock_guard<std::mutex> lock(mutex_);
        x_.reset_data();
        weight_.reset_data();
        bias_.reset_data();
        rng_.reset_data();
    }
    std::string name() const override { return "RofLayerNormBackward"; }
};

Tensor layer_norm_autograd(const Tensor &x, const std::optional<Tensor> &weight_, const std::optional<Tensor> &bias_, double eps,
                           bool relu, double p, const std::optional<Tensor> &rng, int64_t call,
                           std::optional<at::ScalarType> out_type) {
    Tensor out;
    {
        const at::AutoDispatchBelowADInplaceOrView below;
        out = layer_norm_op().call(x, weight_, bias_, eps, relu, p, rng, call, out_type);
    }
    const Tensor weight = weight_.value_or(Tensor()), bias = bias_.value_or(Tensor());
    if (at::GradMode::is_enabled() &&
        (x.requires_grad() || (weight.defined() && weight.requires_grad()) || (bias.defined() && bias.requires_grad()))) {
        auto node = std::shared_ptr<RofLayerNormBackward>(new RofLayerNormBackward(), torch::autograd::deleteNode);
        node->set_next_edges(torch::autograd::collect_next_edges(x, weight, bias));
        node->x_ = SavedVariable(x, false);
        node->weight_ = SavedVariable(weight, false);
        node->bias_ = SavedVariable(bias, false);
        node->rng_ = SavedVariable(p > 0 ? rng.value_or(Tensor()) : Tensor(), false);
        node->eps = eps;
        node->p = p;
        node->relu = relu;
        node->call = call;
        node->out_type = out_type.value_or(x.scalar_type());
        torch::autograd::set_history(out, node);
    }
    return out;
}

// A checkpointed function's second pass runs within the backward pass: its masks would not be the first one's, and the
// gradients wrong.
void check_no_backward() {
    require(torch::autograd::get_current_graph_task_id() == -1,
            "the dropout state cannot move on during a backward pass: a checkpointed function takes the values of next() as an "
            "argument, and a model with dropout_seed is not checkpointed as a whole");
}

// The values of one step, and the state moved on behind it.
Tensor dropout_state_next_cuda(const Tensor &state, int64_t calls) {
    check_no_backward();
    require(state.scalar_type() == at::kLong && state.numel() == 2 && state.is_contiguous() && !state.is_neg(),
            "the dropout state must be a contiguous int64 tensor {seed, offset}");
    require(calls >= 0, "calls must not be negative");
    const c10::DeviceGuard guard(state.device());
    Tensor used = at::empty({2}, state.options());
    check(rof_dropout_state_next((int64_t *)state.data_ptr(), calls, (int64_t *)used.data_ptr(), current_stream(state)),
          "dropout state");
    state.unsafeGetTensorImpl()->bump_version();   // a backward pass that kept the state itself has to notice
    return used;
}

// ---- Python's calls -----------------------------------------------------------------------------------------------
Tensor layer_norm(const Tensor &x, const std::optional<Tensor> &weight, const std::optional<Tensor> &bias, double eps, bool relu,
                  double p, const std::optional<Tensor> &rng, int64_t call, std::optional<at::ScalarType> out_type) {
    check_call(x);
    check_plain(x);
    for (const auto *t : {&weight, &bias, &rng}) check_plain(*t);
    return layer_norm_op().call(x, weight, bias, eps, relu, p, rng, call, out_type);
}
Tensor dropout(const Tensor &x, double p, const std::optional<Tensor> &rng, int64_t call) {
    check_call(x);
    check_plain(x);
    check_plain(rng);
    return dropout_op().call(x, p, rng, call);
}
Tensor dropout_state_next(const Tensor &state, int64_t calls) {
    check_no_backward();
    require(state.is_cuda(), "the dropout state must be on the GPU (move the module there)");
    check_plain(state);
    return dropout_state_next_op().call(state, calls);
}

}  // namespace

TORCH_LIBRARY(rof, m) {
    m.def("layer_norm(Tensor x, Tensor? weight, Tensor? bias, float eps, bool relu, float dropout, Tensor? rng, int call, "
          "ScalarType? out_dtype) -> Tensor");
    m.def("layer_norm_backward(Tensor grad, Tensor x, Tensor? weight, Tensor? bias, float eps, bool relu, float dropout, "
          "Tensor? rng, int call, ScalarType out_dtype, bool want_x, bool want_weight, bool want_bias) -> (Tensor, Tensor, Tensor)");
    m.def("dropout(Tensor x, float p, Tensor? rng, int call) -> Tensor");
    m.def("dropout_state_next(Tensor(a!) state, int calls) -> Tensor");
}
TORCH_LIBRARY_IMPL(rof, CUDA, m) {
    m.impl("layer_norm", &layer_norm_cuda);
    m.impl("layer_norm_backward", &layer_norm_backward_cuda);
    m.impl("dropout", &dropout_cuda);
    m.impl("dropout_state_next", &dropout_state_next_cuda);
}
TORCH_LIBRARY_IMPL(rof, AutogradCUDA, m) {
    m.impl("layer_norm", &layer_norm_autograd);
    m.impl("dropout", &dropout_autograd);
    m.impl("dropout_state_next", torch::CppFunction::makeFallthrough());   // whole numbers
}
// views with the negative bit reach the kernels' checks, which refuse them
TORCH_LIBRARY_IMPL(rof, Negative, m) {
    for (const char *name : {"layer_norm", "layer_norm_backward", "dropout", "dropout_state_next"})
        m.impl(name, torch::CppFunction::makeFallthrough());
}

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
    py::register_exception_translator([](std::exception_ptr p) {
        try {
            if (p) std::rethrow_exception(p);
        } catch (const Failure &e) {
            PyErr_SetString(g_error_type ? g_error_type : PyExc_RuntimeError, e.what());
        }
    });
    m.def("set_error_type", [](py::object type) {
        Py_XDECREF(g_error_type);
        g_error_type = type.release().ptr();
    });
    m.def("layer_norm", &layer_norm, "dropout(relu(layer norm)) of every row (gfx950)");
    m.def("dropout", &dropout, "dropout without a stored mask (gfx950)");
    m.def("dropout_state_next", &dropout_state_next, "the values of one step; moves the state on (gfx950)");
}
