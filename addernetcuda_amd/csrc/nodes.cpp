// The host side of the layers beside the adder layers: arguments, outputs and autograd nodes of linear_act and layer_norm, and the walk over an
// AdamW step's tensors, as a CPython module on top of the C ABI.
//
// A node whose backward is Python costs 50 us a pass on the host (the engine's thread waits for the interpreter), an optimizer step that looks at
// every tensor from Python more than a microsecond a tensor -- as much as or more than these kernels take on all but large tensors.  The module
// is compiled against torch's C++ interface; the kernels stay behind include/addernet_hip.h, whose entry points it is handed by address (bind), so
// that it runs on the library that the package has loaded.
#include <Python.h>

#include <ATen/ops/empty.h>
#include <ATen/ops/zeros.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/python_variable.h>

#include <string>
#include <vector>

#include "../../include/addernet_hip.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::Variable;
using torch::autograd::variable_list;

struct Library {
    decltype(&adder_strerror) strerror_;
    decltype(&adder_last_hip_error) last_hip_error;
    decltype(&adder_linear_fwd_workspace_bytes) linear_fwd_bytes;
    decltype(&adder_linear_fwd) linear_fwd;
    decltype(&adder_linear_bwd_workspace_bytes) linear_bwd_bytes;
    decltype(&adder_linear_bwd) linear_bwd;
    decltype(&adder_layer_norm_fwd) norm_fwd;
    decltype(&adder_layer_norm_bwd_workspace_bytes) norm_bwd_bytes;
    decltype(&adder_layer_norm_bwd) norm_bwd;
    decltype(&adder_adamw_step) adamw;
    decltype(&adder_adamw_step_8bit) adamw8;
    decltype(&adder_adamw_advance) advance;
} lib;

void check(int status, const char *what) {
    if (status == ADDER_OK) return;
    std::string text = lib.strerror_(status);
    if (status == ADDER_ERR_HIP) text += std::string(": ") + lib.last_hip_error();
    TORCH_CHECK(false, what, ": ", text);
}

// The interpreter is free for other threads while this lives: a launch waits where the queue is full
struct Released {
    PyThreadState *const state = PyEval_SaveThread();
    Released() = default;
    Released(const Released &) = delete;
    ~Released() { PyEval_RestoreThread(state); }
};

int type_of(const Tensor &t) { return t.scalar_type() == at::kBFloat16 ? ADDER_TYPE_BF16 : ADDER_TYPE_F32; }
void *stream_of(const Tensor &t) { return c10::hip::getCurrentHIPStream(t.device().index()).stream(); }
void *ptr(const Tensor &t) { return t.defined() ? t.data_ptr() : nullptr; }
Tensor bytes_for(size_t n, const Tensor &like) {
    return n ? at::empty({(int64_t)n}, like.options().dtype(at::kByte)) : Tensor();
}
Tensor filled(bool zeros, at::IntArrayRef shape, const at::TensorOptions &options) {
    return zeros ? at::zeros(shape, options) : at::empty(shape, options);
}
std::string shape_text(at::IntArrayRef s) {   // as Python prints it
    std::string t = "(";
    for (size_t i = 0; i < s.size(); ++i) t += std::to_string(s[i]) + (i + 1 < s.size() ? ", " : s.size() == 1 ? "," : "");
    return t + ")";
}

// t as rows of `width` neighbouring values, and their stride: a view where it is one.  Values of one row lie side by side, and rows that are not all
// the same one do not overlap.
struct Rows { Tensor t; long stride, rows; };
Rows as_rows(const Tensor &t, int64_t width) {
    const int64_t rows = t.numel() / width;
    if (t.is_contiguous()) return {t, (long)width, (long)rows};
    Tensor v = t.dim() == 2 && t.size(1) == width ? t : t.reshape({rows, width});   // (two dimensions may also be one row: all of them normalised)
    if ((width > 1 && v.stride(1) != 1) || (rows > 1 && v.stride(0) < width && v.stride(0) != 0)) v = v.contiguous();
    return {v, rows > 1 ? (long)v.stride(0) : (long)width, (long)rows};
}

// Gradients that these nodes give have no formula to be differentiated again: whoever tries is told so
variable_list once(variable_list grads, const char *what) {
    if (!at::GradMode::is_enabled()) return grads;
    variable_list some;
    for (const auto &g : grads)
        if (g.defined()) some.push_back(g.detach().requires_grad_(true));
    if (some.empty()) return grads;
    auto error = std::make_shared<torch::autograd::DelayedError>(std::string("trying to differentiate twice a function that was marked with once_differentiable: ") + what,
                                                                 (int64_t)some.size());
    auto wrapped = (*error)(std::move(some));
    size_t k = 0;
    for (auto &g : grads)
        if (g.defined()) g = wrapped[k++];
    return grads;
}

// ---- linear layers -----------------------------------------------------------------------------------------------------
Tensor linear_forward(const Tensor &x, const Tensor &w, const Tensor &bias, const Tensor &residual, int64_t act, Tensor *pre) {
    const int64_t n = w.size(0), k = w.size(1);
    c10::SmallVector<int64_t, 6> shape(x.sizes().begin(), x.sizes().end());
    shape.back() = n;
    Tensor y = at::empty(shape, x.options());
    if (pre) *pre = at::empty({x.numel() / k, n}, x.options());
    if (y.numel() == 0) return y;
    const c10::DeviceGuard guard(x.device());
    const Rows a = as_rows(x, k);
    const Rows r = residual.defined() ? as_rows(residual, n) : Rows{Tensor(), 0, 0};
    size_t need = 0;
    const int type = type_of(x);
    check(lib.linear_fwd_bytes(a.rows, (int)k, (int)n, type, &need), "adder_linear_fwd_workspace_bytes");
    const Tensor ws = bytes_for(need, x);
    check(lib.linear_fwd(a.t.data_ptr(), a.stride, w.data_ptr(), ptr(bias), ptr(r.t), r.stride, y.data_ptr(), pre ? pre->data_ptr() : nullptr, (int)act,
                         a.rows, (int)k, (int)n, type, ptr(ws), need, stream_of(x)),
          "adder_linear_fwd");
    return y;
}

// Arguments that may be absent reach a node as optionals; its edges count those that are there
typedef std::optional<Variable> Maybe;
Maybe maybe(const Tensor &t) { return t.defined() ? Maybe(t) : Maybe(); }

struct LinearAct : public torch::autograd::Function<LinearAct> {
    static Variable forward(AutogradContext *ctx, const Variable &x, const Variable &w, const Maybe &has_bias, const Maybe &has_residual, int64_t act) {
        const Tensor bias = has_bias.value_or(Tensor()), residual = has_residual.value_or(Tensor());
        const bool wx = x.requires_grad(), ww = w.requires_grad(), wb = bias.defined() && bias.requires_grad();
        // what the activation's derivative is taken from: the values before it, or ReLU's own result where nothing was added to it
        const bool keep = act != ADDER_ACT_NONE && (wx || ww || wb), own = act == ADDER_ACT_RELU && !residual.defined();
        Tensor pre;
        const Tensor y = linear_forward(x, w, bias, residual, act, keep && !own ? &pre : nullptr);
        if (keep && own) pre = y;
        ctx->save_for_backward({ww ? x : Variable(), wx ? w : Variable(), pre});
        ctx->saved_data["act"] = act;
        ctx->saved_data["x"] = x.sizes().vec();
        ctx->saved_data["n"] = w.size(0);
        ctx->saved_data["bias"] = bias.defined();
        ctx->saved_data["residual"] = residual.defined();
        return y;
    }
    static variable_list backward(AutogradContext *ctx, const variable_list &grads) {
        const auto saved = ctx->get_saved_variables();
        const Tensor &dy = grads[0];
        const bool bias = ctx->saved_data["bias"].toBool(), want_x = ctx->needs_input_grad(0), want_w = ctx->needs_input_grad(1);
        const bool want_b = bias && ctx->needs_input_grad(2), want_r = ctx->saved_data["residual"].toBool() && ctx->needs_input_grad(bias ? 3 : 2);
        variable_list out(5);
        if (!dy.defined()) return out;
        if (want_r) out[3] = dy;
        if (want_x || want_w || want_b) {
            const at::AutoGradMode off(false);
            const int64_t act = ctx->saved_data["act"].toInt(), n = ctx->saved_data["n"].toInt();
            const std::vector<int64_t> x_shape = ctx->saved_data["x"].toIntVector();
            const int64_t k = x_shape.back();
            const bool none = dy.numel() == 0;
            if (want_x) out[0] = filled(none, x_shape, dy.options());
            if (want_w) out[1] = filled(none, {n, k}, dy.options());
            if (want_b) out[2] = filled(none, {n}, dy.options());
            if (!none) {
                const c10::DeviceGuard guard(dy.device());
                const Rows d = as_rows(dy, n);
                const Rows x = want_w ? as_rows(saved[0], k) : Rows{Tensor(), (long)k, 0};
                size_t need = 0;
                const int type = type_of(dy);
                check(lib.linear_bwd_bytes(d.rows, (int)k, (int)n, (int)act, type, &need), "adder_linear_bwd_workspace_bytes");
                const Tensor ws = bytes_for(need, dy);
                check(lib.linear_bwd(d.t.data_ptr(), d.stride, ptr(saved[2]), ptr(x.t), x.stride, ptr(saved[1]), ptr(out[0]), ptr(out[1]), ptr(out[2]),
                                     (int)act, d.rows, (int)k, (int)n, type, ptr(ws), need, stream_of(dy)),
                      "adder_linear_bwd");
            }
        }
        return once(std::move(out), "linear_act");
    }
};

Tensor optional_tensor(PyObject *o, const char *name) {
    if (o == Py_None) return Tensor();
    if (!THPVariable_Check(o)) throw torch::TypeError(std::string(name) + " must be a torch.Tensor");
    return THPVariable_Unpack(o);
}

// linear_act(x, weight, bias or None, residual or None, act): all plain GPU tensors, x float32 or bfloat16, no empty weight
PyObject *py_linear_act(PyObject *, PyObject *const *args, Py_ssize_t count) {
    HANDLE_TH_ERRORS
    TORCH_CHECK(count == 5, "linear_act: five arguments");
    const Tensor x = optional_tensor(args[0], "x");
    Tensor w = optional_tensor(args[1], "weight"), bias = optional_tensor(args[2], "bias"), residual = optional_tensor(args[3], "residual");
    const int64_t act = PyLong_AsLong(args[4]);
    TORCH_CHECK(w.dim() == 2, "weight must have two dimensions, got ", shape_text(w.sizes()));
    const int64_t n = w.size(0), k = w.size(1);
    TORCH_CHECK(x.dim() > 0 && x.size(-1) == k, "x has shape ", shape_text(x.sizes()), " but the weight expects ", k, " features");
    TORCH_CHECK(!bias.defined() || (bias.dim() == 1 && bias.size(0) == n), "bias must have shape (", n, ",), got ", shape_text(bias.sizes()));
    for (const Tensor *t : {&w, &bias, &residual}) {
        if (!t->defined()) continue;
        TORCH_CHECK(t->device() == x.device(), "all tensors must be on the same device");
        TORCH_CHECK(t->scalar_type() == x.scalar_type(), "all tensors must have the type of x, ", x.dtype(), ", got ", t->dtype());
    }
    if (residual.defined()) {
        c10::SmallVector<int64_t, 6> shape(x.sizes().begin(), x.sizes().end());
        shape.back() = n;
        if (residual.sizes() != at::IntArrayRef(shape)) {
            bool fits = residual.dim() <= (int64_t)shape.size();
            for (int64_t i = 1; fits && i <= residual.dim(); ++i) fits = residual.size(-i) == 1 || residual.size(-i) == shape[shape.size() - i];
            TORCH_CHECK(fits, "residual of shape ", shape_text(residual.sizes()), " does not broadcast to ", shape_text(shape));
            residual = residual.expand(shape);
        }
    }
    Tensor y;
    {
        const Released released;
        w = w.contiguous();
        if (bias.defined()) bias = bias.contiguous();
        const bool grad = at::GradMode::is_enabled() && (x.requires_grad() || w.requires_grad() || (bias.defined() && bias.requires_grad()) ||
                                                         (residual.defined() && residual.requires_grad()));
        y = grad ? LinearAct::apply(x, w, maybe(bias), maybe(residual), act) : linear_forward(x, w, bias, residual, act, nullptr);
    }
    return THPVariable_Wrap(std::move(y));
    END_HANDLE_TH_ERRORS
}

// ---- layer normalisation -------------------------------------------------------------------------------------------------
Tensor norm_forward(const Tensor &x, const Tensor &weight, const Tensor &bias, int64_t width, double eps, Tensor *mean, Tensor *rstd) {
    Tensor y = at::empty(x.sizes(), x.options());
    const int64_t rows = x.numel() / width;
    if (mean) {
        *mean = at::empty({rows}, x.options().dtype(at::kFloat));
        *rstd = at::empty({rows}, x.options().dtype(at::kFloat));
    }
    if (rows == 0) return y;
    const c10::DeviceGuard guard(x.device());
    const Rows a = as_rows(x, width);
    const Tensor &of = weight.defined() ? weight : bias.defined() ? bias : x;
    check(lib.norm_fwd(a.t.data_ptr(), a.stride, ptr(weight), ptr(bias), y.data_ptr(), mean ? mean->data_ptr<float>() : nullptr,
                       mean ? rstd->data_ptr<float>() : nullptr, (float)eps, a.rows, (int)width, type_of(x), type_of(of), stream_of(x)),
          "adder_layer_norm_fwd");
    return y;
}

struct LayerNorm : public torch::autograd::Function<LayerNorm> {
    static Variable forward(AutogradContext *ctx, const Variable &x, const Maybe &has_weight, const Maybe &has_bias, int64_t width, double eps) {
        const Tensor weight = has_weight.value_or(Tensor()), bias = has_bias.value_or(Tensor());
        Tensor mean, rstd;
        const Tensor y = norm_forward(x, weight, bias, width, eps, &mean, &rstd);
        ctx->save_for_backward({x, weight, bias.defined() && bias.requires_grad() ? bias : Variable(), mean, rstd});
        ctx->saved_data["width"] = width;
        ctx->saved_data["bias"] = bias.defined();
        ctx->saved_data["type"] = (int64_t)type_of(weight.defined() ? weight : bias.defined() ? bias : x);
        return y;
    }
    static variable_list backward(AutogradContext *ctx, const variable_list &grads) {
        const auto saved = ctx->get_saved_variables();
        const Tensor &dy = grads[0], &x = saved[0], &weight = saved[1], &bias = saved[2];
        const bool want_x = ctx->needs_input_grad(0), want_w = weight.defined() && ctx->needs_input_grad(1);
        const bool want_b = ctx->saved_data["bias"].toBool() && ctx->needs_input_grad(weight.defined() ? 2 : 1);
        variable_list out(5);
        if (!dy.defined()) return out;
        {
            const at::AutoGradMode off(false);
            const int64_t width = ctx->saved_data["width"].toInt();
            const bool none = dy.numel() == 0;
            if (want_x) out[0] = filled(none, x.sizes(), x.options());
            if (want_w) out[1] = filled(none, weight.sizes(), weight.options());
            if (want_b) out[2] = filled(none, bias.sizes(), bias.options());
            if (!none) {
                const c10::DeviceGuard guard(dy.device());
                const Rows a = as_rows(x, width), d = as_rows(dy, width);
                size_t need = 0;
                const int type = type_of(x);
                if (want_w || want_b) check(lib.norm_bwd_bytes(a.rows, (int)width, type, &need), "adder_layer_norm_bwd_workspace_bytes");
                const Tensor ws = bytes_for(need, x);
                check(lib.norm_bwd(d.t.data_ptr(), d.stride, a.t.data_ptr(), a.stride, ptr(weight), saved[3].data_ptr<float>(), saved[4].data_ptr<float>(),
                                   ptr(out[0]), ptr(out[1]), ptr(out[2]), a.rows, (int)width, type, (int)ctx->saved_data["type"].toInt(), ptr(ws), need,
                                   stream_of(x)),
                      "adder_layer_norm_bwd");
            }
        }
        return once(std::move(out), "layer_norm");
    }
};

// layer_norm(x, weight or None, bias or None, eps): as above, and no empty last dimensions
PyObject *py_layer_norm(PyObject *, PyObject *const *args, Py_ssize_t count) {
    HANDLE_TH_ERRORS
    TORCH_CHECK(count == 4, "layer_norm: four arguments");
    const Tensor x = optional_tensor(args[0], "x");
    Tensor weight = optional_tensor(args[1], "weight"), bias = optional_tensor(args[2], "bias");
    const double eps = PyFloat_AsDouble(args[3]);
    if (PyErr_Occurred()) return nullptr;
    TORCH_CHECK(eps >= 0, "eps must not be negative, got ", eps);
    const Tensor &of = weight.defined() ? weight : bias;
    const at::IntArrayRef shape = of.defined() ? of.sizes() : x.sizes().slice(x.dim() ? x.dim() - 1 : 0);
    const int64_t dims = (int64_t)shape.size();
    TORCH_CHECK(dims > 0 && x.dim() >= dims && x.sizes().slice(x.dim() - dims) == shape, "x has shape ", shape_text(x.sizes()),
                " but the last dimensions are to be ", shape_text(shape));
    for (const Tensor *t : {&weight, &bias}) {
        if (!t->defined()) continue;
        const char *name = t == &weight ? "weight" : "bias";
        TORCH_CHECK(t->sizes() == shape, name, " must have shape ", shape_text(shape), ", got ", shape_text(t->sizes()));
        TORCH_CHECK(t->device() == x.device(), "all tensors must be on the same device");
        TORCH_CHECK(t->scalar_type() == of.scalar_type() &&
                        (t->scalar_type() == x.scalar_type() || (x.scalar_type() == at::kBFloat16 && t->scalar_type() == at::kFloat)),
                    name, " must have the type of x (or float32 beside bfloat16), ", x.dtype(), ", got ", t->dtype());
    }
    int64_t width = 1;
    for (const int64_t d : shape) width *= d;
    Tensor y;
    {
        const Released released;
        if (weight.defined()) weight = weight.contiguous();
        if (bias.defined()) bias = bias.contiguous();
        const bool grad = at::GradMode::is_enabled() && (x.requires_grad() || (weight.defined() && weight.requires_grad()) || (bias.defined() && bias.requires_grad()));
        y = grad ? LayerNorm::apply(x, maybe(weight), maybe(bias), width, eps) : norm_forward(x, weight, bias, width, eps, nullptr, nullptr);
    }
    return THPVariable_Wrap(std::move(y));
    END_HANDLE_TH_ERRORS
}

// ---- AdamW ------------------------------------------------------------------------------------------------------------------
constexpr int64_t kPieceMost = (int64_t)1 << 30;   // values of one entry of the kernel's table; longer tensors take several

struct Batch {   // what one step count, storage type of the parameter and of its state have in common
    long count;              // of this step
    float *step;             // capturable: where it is counted
    at::ScalarType type;
    bool coded;
    std::vector<void *> p, g, m, v, ms, vs;
    std::vector<long> n;
};

struct Held {   // references to objects, while this lives
    std::vector<PyObject *> objects;
    Held() = default;
    Held(const Held &) = delete;
    void add(PyObject *o) {
        objects.push_back(o);
        Py_INCREF(o);
    }
    ~Held() {
        for (PyObject *o : objects) Py_DECREF(o);
    }
};

PyObject *key(const char *name) { return PyUnicode_InternFromString(name); }

// adamw_step(params, states, capturable, lr, lr_device, beta1, beta2, eps, weight_decay, piece, groups): one step of parameters with gradients, with their
// states (dicts).  False, and nothing done, where a parameter, a gradient or a state is not what the kernels take; an error where a state does not
// fit its parameter.
PyObject *py_adamw_step(PyObject *, PyObject *const *args, Py_ssize_t count) {
    HANDLE_TH_ERRORS
    TORCH_CHECK(count == 11, "adamw_step: eleven arguments");
    static PyObject *const names[] = {key("step"), key("exp_avg"), key("exp_avg_sq"), key("exp_avg_scale"), key("exp_avg_sq_scale")};
    PyObject *params = args[0], *states = args[1];
    TORCH_CHECK(PyList_Check(params) && PyList_Check(states) && PyList_GET_SIZE(params) == PyList_GET_SIZE(states), "adamw_step: two lists");
    const bool capturable = PyObject_IsTrue(args[2]);
    const double lr = PyFloat_AsDouble(args[3]);
    const float *lr_device = reinterpret_cast<const float *>(PyLong_AsSize_t(args[4]));
    const double b1 = PyFloat_AsDouble(args[5]), b2 = PyFloat_AsDouble(args[6]), eps = PyFloat_AsDouble(args[7]), decay = PyFloat_AsDouble(args[8]);
    const int64_t piece = PyLong_AsLongLong(args[9]), groups = PyLong_AsLongLong(args[10]);
    if (PyErr_Occurred()) return nullptr;
    TORCH_CHECK(piece > 0 && piece <= kPieceMost && piece % ADDER_STATE_BLOCK == 0, "adamw_step: pieces of whole blocks");
    const Py_ssize_t all = PyList_GET_SIZE(params);
    std::vector<Batch> batches;
    Held held;   // what another thread could replace before it is launched: the states' tensors and the gradients
    std::vector<Tensor> gradients;
    held.objects.reserve(5 * all);
    std::vector<long> counts;   // of this step
    gradients.reserve(all);
    counts.reserve(all);
    c10::Device device(c10::DeviceType::CPU);
    for (Py_ssize_t i = 0; i < all; ++i) {
        PyObject *po = PyList_GET_ITEM(params, i), *so = PyList_GET_ITEM(states, i);
        if (!THPVariable_Check(po) || !PyDict_Check(so)) Py_RETURN_FALSE;
        const Tensor &p = THPVariable_Unpack(po);
        const Tensor &g = p.grad();
        if (i == 0) device = p.device();
        const at::ScalarType type = p.scalar_type();
        if (!g.defined() || !p.is_cuda() || p.device() != device || g.device() != device || (type != at::kFloat && type != at::kBFloat16) ||
            g.scalar_type() != type || g.layout() != at::kStrided || p.layout() != at::kStrided || !p.is_contiguous() || !g.is_contiguous() ||
            g.numel() != p.numel())
            Py_RETURN_FALSE;
        PyObject *items[5];
        for (int k = 0; k < 3; ++k) items[k] = PyDict_GetItem(so, names[k]);
        if (!items[0] || !items[1] || !items[2] || !THPVariable_Check(items[1]) || !THPVariable_Check(items[2])) Py_RETURN_FALSE;
        const Tensor &m = THPVariable_Unpack(items[1]), &v = THPVariable_Unpack(items[2]);
        const bool coded = m.scalar_type() == at::kChar;
        if (!coded && (m.scalar_type() != at::kFloat || v.scalar_type() != at::kFloat)) Py_RETURN_FALSE;
        long step_count = 0;
        float *step = nullptr;
        if (capturable) {
            if (!THPVariable_Check(items[0])) Py_RETURN_FALSE;
            const Tensor &t = THPVariable_Unpack(items[0]);
            if (t.device() != device || t.scalar_type() != at::kFloat || t.numel() != 1) Py_RETURN_FALSE;
            step = t.data_ptr<float>();
        } else {
            if (!PyLong_CheckExact(items[0])) Py_RETURN_FALSE;
            step_count = PyLong_AsLong(items[0]) + 1;
        }
        const int64_t n = p.numel();
        const auto fits = [&](const Tensor &t, at::ScalarType want, int64_t values) {
            TORCH_CHECK(t.scalar_type() == want && t.numel() == values && t.is_contiguous() && t.device() == device,
                        "adamw_step: the state does not fit its parameter");
        };
        fits(m, coded ? at::kChar : at::kFloat, n);
        fits(v, coded ? at::kByte : at::kFloat, n);
        gradients.push_back(g);
        counts.push_back(step_count);
        for (int k = 0; k < 3; ++k) held.add(items[k]);
        Tensor ms, vs;
        if (coded) {
            for (int k = 3; k < 5; ++k) items[k] = PyDict_GetItem(so, names[k]);
            TORCH_CHECK(items[3] && items[4] && THPVariable_Check(items[3]) && THPVariable_Check(items[4]), "adamw_step: the state does not fit its parameter");
            ms = THPVariable_Unpack(items[3]);
            vs = THPVariable_Unpack(items[4]);
            fits(ms, at::kFloat, (n + ADDER_STATE_BLOCK - 1) / ADDER_STATE_BLOCK);
            fits(vs, at::kFloat, (n + ADDER_STATE_BLOCK - 1) / ADDER_STATE_BLOCK);
            for (int k = 3; k < 5; ++k) held.add(items[k]);
        }
        Batch *batch = nullptr;
        for (Batch &b : batches)
            if (b.count == step_count && b.step == step && b.type == type && b.coded == coded) batch = &b;
        if (!batch) {
            batches.push_back(Batch{step_count, step, type, coded, {}, {}, {}, {}, {}, {}, {}});
            batch = &batches.back();
            for (auto *to : {&batch->p, &batch->g, &batch->m, &batch->v}) to->reserve(all - i);
            batch->n.reserve(all - i);
        }
        const int64_t size = type == at::kFloat ? 4 : 2, state = coded ? 1 : 4;
        for (int64_t at = 0; at < n; at += piece) {   // (empty tensors have no entry)
            const auto in = [at](const Tensor &t, int64_t each) { return static_cast<char *>(t.data_ptr()) + at * each; };
            batch->p.push_back(in(p, size));
            batch->g.push_back(in(g, size));
            batch->m.push_back(in(m, state));
            batch->v.push_back(in(v, state));
            if (coded) {
                batch->ms.push_back(ms.data_ptr<float>() + at / ADDER_STATE_BLOCK);
                batch->vs.push_back(vs.data_ptr<float>() + at / ADDER_STATE_BLOCK);
            }
            batch->n.push_back((long)(n - at < piece ? n - at : piece));
        }
    }
    if (all == 0) Py_RETURN_TRUE;
    {
        const Released released;
        const c10::DeviceGuard guard(device);
        void *stream = c10::hip::getCurrentHIPStream(device.index()).stream();
        std::vector<std::pair<float *, Tensor>> advanced;
        for (const Batch &b : batches) {
            const float *corr = nullptr;
            if (capturable) {
                for (const auto &a : advanced)
                    if (a.first == b.step) corr = a.second.data_ptr<float>();
                if (!corr) {
                    advanced.emplace_back(b.step, at::empty({2}, at::TensorOptions().dtype(at::kFloat).device(device)));
                    float *to = advanced.back().second.data_ptr<float>();
                    check(lib.advance(b.step, b1, b2, to, stream), "adder_adamw_advance");
                    corr = to;
                }
            }
            const int type = b.type == at::kFloat ? ADDER_TYPE_F32 : ADDER_TYPE_BF16;
            const size_t most = b.coded ? ADDER_ADAMW_8BIT_BATCH_MAX : ADDER_ADAMW_BATCH_MAX;
            for (size_t i = 0, next; i < b.n.size(); i = next) {   // as many as a table holds and a launch has workgroups for
                int64_t used = 0;
                for (next = i; next < b.n.size() && next - i < most; ++next) {
                    used += (b.n[next] + 1023) / 1024;
                    if (next > i && used > groups) break;
                }
                const int k = (int)(next - i);
                const void *const *g = const_cast<const void *const *>(b.g.data() + i);
                if (b.coded)
                    check(lib.adamw8(k, b.p.data() + i, g, reinterpret_cast<signed char *const *>(b.m.data() + i),
                                     reinterpret_cast<unsigned char *const *>(b.v.data() + i), reinterpret_cast<float *const *>(b.ms.data() + i),
                                     reinterpret_cast<float *const *>(b.vs.data() + i), b.n.data() + i, lr_device, lr, b1, b2, eps, decay, b.count, corr, type,
                                     stream),
                          "adder_adamw_step_8bit");
                else
                    check(lib.adamw(k, b.p.data() + i, g, reinterpret_cast<float *const *>(b.m.data() + i), reinterpret_cast<float *const *>(b.v.data() + i),
                                    b.n.data() + i, lr_device, lr, b1, b2, eps, decay, b.count, corr, type, stream),
                          "adder_adamw_step");
            }
        }
    }
    PyObject *next = nullptr;
    long of = -1;
    for (Py_ssize_t i = 0; i < all; ++i) {
        THPVariable_Unpack(PyList_GET_ITEM(params, i)).unsafeGetTensorImpl()->bump_version();   // (changed in place)
        if (capturable) continue;
        PyObject *so = PyList_GET_ITEM(states, i);
        const long now = counts[i];
        if (now != of) {
            Py_XDECREF(next);
            next = PyLong_FromLong(of = now);
        }
        if (PyDict_SetItem(so, names[0], next)) {
            Py_XDECREF(next);
            return nullptr;
        }
    }
    Py_XDECREF(next);
    Py_RETURN_TRUE;
    END_HANDLE_TH_ERRORS
}

// bind({name: address}): the entry points of the loaded library
PyObject *py_bind(PyObject *, PyObject *names) {
    HANDLE_TH_ERRORS
    const auto take = [names](const char *name, auto &to) {
        PyObject *o = PyDict_GetItemString(names, name);
        TORCH_CHECK(o, "bind: no ", name);
        to = reinterpret_cast<std::remove_reference_t<decltype(to)>>(PyLong_AsSize_t(o));
    };
    take("adder_strerror", lib.strerror_);
    take("adder_last_hip_error", lib.last_hip_error);
    take("adder_linear_fwd_workspace_bytes", lib.linear_fwd_bytes);
    take("adder_linear_fwd", lib.linear_fwd);
    take("adder_linear_bwd_workspace_bytes", lib.linear_bwd_bytes);
    take("adder_linear_bwd", lib.linear_bwd);
    take("adder_layer_norm_fwd", lib.norm_fwd);
    take("adder_layer_norm_bwd_workspace_bytes", lib.norm_bwd_bytes);
    take("adder_layer_norm_bwd", lib.norm_bwd);
    take("adder_adamw_step", lib.adamw);
    take("adder_adamw_step_8bit", lib.adamw8);
    take("adder_adamw_advance", lib.advance);
    if (PyErr_Occurred()) return nullptr;
    Py_RETURN_NONE;
    END_HANDLE_TH_ERRORS
}

PyMethodDef methods[] = {
    {"bind", py_bind, METH_O, nullptr},
    {"linear_act", reinterpret_cast<PyCFunction>(reinterpret_cast<void *>(py_linear_act)), METH_FASTCALL, nullptr},
    {"layer_norm", reinterpret_cast<PyCFunction>(reinterpret_cast<void *>(py_layer_norm)), METH_FASTCALL, nullptr},
    {"adamw_step", reinterpret_cast<PyCFunction>(reinterpret_cast<void *>(py_adamw_step)), METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr},
};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_nodes", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__nodes() { return PyModule_Create(&module); }
