// The host side of gated blocks, their 8-bit form and their training from a teacher: arguments, outputs and autograd nodes of rms_norm,
// gated_linear, the 8-bit products and the loss against a teacher's logits.
#include "nodes.hpp"

namespace nodes {
namespace {

int64_t blocks_of(int64_t n) { return (n + ADDER_CODE_BLOCK - 1) / ADDER_CODE_BLOCK; }
bool wants_grad(const Tensor &t) { return t.defined() && t.requires_grad(); }
double number(PyObject *o) {
    const double v = PyFloat_AsDouble(o);
    if (v == -1.0 && PyErr_Occurred()) throw python_error();
    return v;
}
int64_t integer(PyObject *o) {
    const int64_t v = PyLong_AsLongLong(o);
    if (v == -1 && PyErr_Occurred()) throw python_error();
    return v;
}
// what codes are made of, or added to, has no gradient through them
void no_gradients(const char *what, std::initializer_list<const Tensor *> all) {
    if (!at::GradMode::is_enabled()) return;
    for (const Tensor *t : all) TORCH_CHECK(!wants_grad(*t), what, " has no gradient: call it under torch.no_grad(), or on detached tensors");
}
// residual as a tensor of `shape`
Tensor expanded(const Tensor &residual, at::IntArrayRef shape) {
    if (residual.sizes() == shape) return residual;
    bool fits = residual.dim() <= (int64_t)shape.size();
    for (int64_t i = 1; fits && i <= residual.dim(); ++i) fits = residual.size(-i) == 1 || residual.size(-i) == shape[shape.size() - i];
    TORCH_CHECK(fits, "residual of shape ", shape_text(residual.sizes()), " does not broadcast to ", shape_text(shape));
    return residual.expand(shape);
}

// ---- RMS norm ------------------------------------------------------------------------------------------------------------
struct Normed { Tensor y, scale, sum, rstd; };
Normed rms_forward(const Tensor &x, const Tensor &weight, const Tensor &residual, double eps, bool codes, bool keep) {
    Normed out;
    const int64_t width = x.size(-1), rows = width ? x.numel() / width : 0;
    out.y = at::empty(x.sizes(), codes ? x.options().dtype(at::kFloat8_e4m3fn) : x.options());
    if (codes) {
        c10::SmallVector<int64_t, 6> shape(x.sizes().begin(), x.sizes().end());
        shape.back() = blocks_of(width);
        out.scale = at::empty(shape, x.options().dtype(at::kFloat));
    }
    if (residual.defined()) out.sum = at::empty(x.sizes(), x.options());
    if (keep) out.rstd = at::empty({rows}, x.options().dtype(at::kFloat));
    if (rows == 0) return out;
    const c10::DeviceGuard guard(x.device());
    const Rows a = as_rows(x, width), r = residual.defined() ? as_rows(residual, width) : Rows{Tensor(), 0, 0};
    const int type = type_of(x), weight_type = type_of(weight.defined() ? weight : x);
    if (codes)
        check(lib.rms_fwd_codes(a.t.data_ptr(), a.stride, ptr(r.t), r.stride, ptr(weight), ptr(out.sum), static_cast<unsigned char *>(out.y.data_ptr()),
                                out.scale.data_ptr<float>(), (float)eps, rows, (int)width, type, weight_type, stream_of(x)),
              "adder_rms_norm_fwd_codes");
    else
        check(lib.rms_fwd(a.t.data_ptr(), a.stride, ptr(r.t), r.stride, ptr(weight), ptr(out.sum), out.y.data_ptr(),
                          keep ? out.rstd.data_ptr<float>() : nullptr, (float)eps, rows, (int)width, type, weight_type, stream_of(x)),
              "adder_rms_norm_fwd");
    return out;
}

struct RmsNorm : public torch::autograd::Function<RmsNorm> {
    static variable_list forward(AutogradContext *ctx, const Variable &x, const Maybe &has_weight, const Maybe &has_residual, double eps) {
        const Tensor weight = has_weight.value_or(Tensor()), residual = has_residual.value_or(Tensor());
        const Normed n = rms_forward(x, weight, residual, eps, false, true);
        ctx->set_materialize_grads(false);
        ctx->save_for_backward({residual.defined() ? n.sum : x, weight, n.rstd});
        ctx->saved_data["weight"] = weight.defined();
        ctx->saved_data["residual"] = residual.defined();
        return residual.defined() ? variable_list{n.y, n.sum} : variable_list{n.y};
    }
    static variable_list backward(AutogradContext *ctx, const variable_list &grads) {
        refuse_in_capture("rms_norm");
        const auto saved = ctx->get_saved_variables();
        const Tensor &s = saved[0], &weight = saved[1], &rstd = saved[2];
        const bool has_w = ctx->saved_data["weight"].toBool(), has_r = ctx->saved_data["residual"].toBool();
        const Tensor dy = grads[0], ds = has_r ? grads[1] : Tensor();
        const bool want_x = ctx->needs_input_grad(0), want_w = has_w && ctx->needs_input_grad(1), want_r = has_r && ctx->needs_input_grad(has_w ? 2 : 1);
        variable_list out(4);
        {
            const at::AutoGradMode off(false);
            Tensor gx;
            if (!dy.defined()) {
                gx = ds;
            } else {
                const int64_t width = s.size(-1);
                const bool none = dy.numel() == 0;
                if (want_x || want_r) gx = filled(none, s.sizes(), s.options());
                if (want_w) out[1] = filled(none, weight.sizes(), weight.options());
                if (!none && (gx.defined() || want_w)) {
                    const c10::DeviceGuard guard(s.device());
                    const Rows a = as_rows(s, width), d = as_rows(dy, width), e = ds.defined() ? as_rows(ds, width) : Rows{Tensor(), 0, 0};
                    size_t need = 0;
                    const int type = type_of(s);
                    if (want_w) check(lib.rms_bwd_bytes(a.rows, (int)width, type, &need), "adder_rms_norm_bwd_workspace_bytes");
                    const Tensor ws = bytes_for(need, s);
                    check(lib.rms_bwd(d.t.data_ptr(), d.stride, ptr(e.t), e.stride, a.t.data_ptr(), a.stride, ptr(weight), rstd.data_ptr<float>(), ptr(gx),
                                      ptr(out[1]), a.rows, (int)width, type, type_of(has_w ? weight : s), ptr(ws), need, stream_of(s)),
                          "adder_rms_norm_bwd");
                }
            }
            if (want_x) out[0] = gx;
            if (want_r) out[2] = gx;
        }
        return once(std::move(out), "rms_norm");
    }
};

struct NormCall { Tensor x, weight, residual; double eps; };
NormCall norm_call(PyObject *const *args, Py_ssize_t count, const char *what) {
    TORCH_CHECK(count == 4, what, ": four arguments");
    NormCall c{optional_tensor(args[0], "x"), optional_tensor(args[1], "weight"), optional_tensor(args[3], "residual"), number(args[2])};
    TORCH_CHECK(c.eps >= 0, "eps must not be negative, got ", c.eps);
    TORCH_CHECK(c.x.dim() > 0, "x must have a dimension");
    TORCH_CHECK(!c.weight.defined() || (c.weight.dim() == 1 && c.weight.size(0) == c.x.size(-1)), "weight must have shape (", c.x.size(-1), ",), got ",
                shape_text(c.weight.sizes()));
    for (const Tensor *t : {&c.weight, &c.residual}) TORCH_CHECK(!t->defined() || t->device() == c.x.device(), "all tensors must be on the same device");
    TORCH_CHECK(!c.weight.defined() || c.weight.scalar_type() == c.x.scalar_type() || (c.x.scalar_type() == at::kBFloat16 && c.weight.scalar_type() == at::kFloat),
                "weight must have the type of x (or float32 beside bfloat16), ", c.x.dtype(), ", got ", c.weight.dtype());
    TORCH_CHECK(!c.residual.defined() || c.residual.scalar_type() == c.x.scalar_type(), "residual must have the type of x, ", c.x.dtype(), ", got ",
                c.residual.dtype());
    return c;
}

PyObject *pair(const Tensor &a, const Tensor &b, const Tensor &c = Tensor()) {
    const bool three = c.defined();
    PyObject *t = PyTuple_New(three ? 3 : 2);
    if (!t) throw python_error();
    PyTuple_SET_ITEM(t, 0, THPVariable_Wrap(a));
    PyTuple_SET_ITEM(t, 1, THPVariable_Wrap(b));
    if (three) PyTuple_SET_ITEM(t, 2, THPVariable_Wrap(c));
    return t;
}

// rms_norm(x, weight or None, eps, residual or None): plain GPU tensors, x float32 or bfloat16 -> y, or (y, x + residual)
PyObject *py_rms_norm(PyObject *, PyObject *const *args, Py_ssize_t count) {
    HANDLE_TH_ERRORS
    NormCall c = norm_call(args, count, "rms_norm");
    variable_list out;
    {
        const Released released;
        if (c.weight.defined()) c.weight = c.weight.contiguous();
        if (c.residual.defined()) c.residual = expanded(c.residual, c.x.sizes());
        if (at::GradMode::is_enabled() && (wants_grad(c.x) || wants_grad(c.weight) || wants_grad(c.residual))) {
            out = RmsNorm::apply(c.x, maybe(c.weight), maybe(c.residual), c.eps);
        } else {
            const Normed n = rms_forward(c.x, c.weight, c.residual, c.eps, false, false);
            out = {n.y, n.sum};
        }
    }
    return c.residual.defined() ? pair(out[0], out[1]) : THPVariable_Wrap(out[0]);
    END_HANDLE_TH_ERRORS
}

// rms_norm_fp8(x, weight or None, eps, residual or None) -> (codes, scales), and x + residual
PyObject *py_rms_norm_fp8(PyObject *, PyObject *const *args, Py_ssize_t count) {
    HANDLE_TH_ERRORS
    NormCall c = norm_call(args, count, "rms_norm_fp8");
    no_gradients("rms_norm_fp8", {&c.x, &c.weight, &c.residual});
    Normed n;
    {
        const Released released;
        if (c.weight.defined()) c.weight = c.weight.contiguous();
        if (c.residual.defined()) c.residual = expanded(c.residual, c.x.sizes());
        n = rms_forward(c.x, c.weight, c.residual, c.eps, true, false);
    }
    return pair(n.y, n.scale, n.sum);
    END_HANDLE_TH_ERRORS
}

// ---- codes ----------------------------------------------------------------------------------------------------------------
// quantize(x, act or -1) -> (codes, scales)
PyObject *py_quantize(PyObject *, PyObject *const *args, Py_ssize_t count) {
    HANDLE_TH_ERRORS
    TORCH_CHECK(count == 2, "quantize: two arguments");
    const Tensor x = optional_tensor(args[0], "x");
    const int64_t act = integer(args[1]);
    TORCH_CHECK(x.dim() > 0 && (act < 0 || x.size(-1) % 2 == 0), "x must have a last dimension", act < 0 ? "" : " of two halves", ", got ", shape_text(x.sizes()));
    no_gradients("quantize", {&x});
    Tensor q, scale;
    {
        const Released released;
        const int64_t in = x.size(-1), width = act < 0 ? in : in / 2, rows = in ? x.numel() / in : 0;
        c10::SmallVector<int64_t, 6> shape(x.sizes().begin(), x.sizes().end());
        shape.back() = width;
        q = at::empty(shape, x.options().dtype(at::kFloat8_e4m3fn));
        shape.back() = blocks_of(width);
        scale = at::empty(shape, x.options().dtype(at::kFloat));
        if (rows) {
            const c10::DeviceGuard guard(x.device());
            const Rows a = as_rows(x, in);
            check(lib.quantize(a.t.data_ptr(), a.stride, (int)act, static_cast<unsigned char *>(q.data_ptr()), scale.data_ptr<float>(), rows, (int)width,
                               type_of(x), stream_of(x)),
                  "adder_quantize");
        }
    }
    return pair(q, scale);
    END_HANDLE_TH_ERRORS
}

// quantize_weight(w) -> (codes, scales)
PyObject *py_quantize_weight(PyObject *, PyObject *const *args, Py_ssize_t count) {
    HANDLE_TH_ERRORS
    TORCH_CHECK(count == 1, "quantize_weight: one argument");
    const Tensor w = optional_tensor(args[0], "weight");
    TORCH_CHECK(w.dim() == 2 && w.numel() > 0, "weight must have two dimensions that are not empty, got ", shape_text(w.sizes()));
    no_gradients("quantize_weight", {&w});
    Tensor q, scale;
    {
        const Released released;
        const int64_t n = w.size(0), k = w.size(1);
        q = at::empty({n, k}, w.options().dtype(at::kFloat8_e4m3fn));
        scale = at::empty({blocks_of(n), blocks_of(k)}, w.options().dtype(at::kFloat));
        const c10::DeviceGuard guard(w.device());
        const Rows a = as_rows(w, k);
        check(lib.quantize_weight(a.t.data_ptr(), a.stride, static_cast<unsigned char *>(q.data_ptr()), scale.data_ptr<float>(), n, (int)k, type_of(w), stream_of(w)),
              "adder_quantize_weight");
    }
    return pair(q, scale);
    END_HANDLE_TH_ERRORS
}

// linear_fp8(x, x_scale, weight, weight_scale, bias or None, residual or None, act, bfloat16: 1 / float32: 0)
PyObject *py_linear_fp8(PyObject *, PyObject *const *args, Py_ssize_t count) {
    HANDLE_TH_ERRORS
    TORCH_CHECK(count == 8, "linear_fp8: eight arguments");
    Tensor x = optional_tensor(args[0], "x"), xs = optional_tensor(args[1], "x_scale"), w = optional_tensor(args[2], "weight"), ws = optional_tensor(args[3], "weight_scale");
    Tensor bias = optional_tensor(args[4], "bias"), residual = optional_tensor(args[5], "residual");
    const int act = (int)integer(args[6]), type = (int)integer(args[7]);
    const at::ScalarType dtype = type == ADDER_TYPE_BF16 ? at::kBFloat16 : at::kFloat;
    TORCH_CHECK(w.dim() == 2 && w.numel() > 0, "weight must have two dimensions that are not empty, got ", shape_text(w.sizes()));
    const int64_t n = w.size(0), k = w.size(1), blocks = blocks_of(k);
    TORCH_CHECK(x.dim() > 0 && x.size(-1) == k, "x has shape ", shape_text(x.sizes()), " but the weight expects ", k, " features");
    TORCH_CHECK(x.scalar_type() == at::kFloat8_e4m3fn && w.scalar_type() == at::kFloat8_e4m3fn, "x and weight must be float8_e4m3fn, got ", x.dtype(), " and ", w.dtype());
    TORCH_CHECK(xs.scalar_type() == at::kFloat && ws.scalar_type() == at::kFloat, "scales must be float32, got ", xs.dtype(), " and ", ws.dtype());
    c10::SmallVector<int64_t, 6> shape(x.sizes().begin(), x.sizes().end());
    shape.back() = blocks;
    TORCH_CHECK(xs.sizes() == at::IntArrayRef(shape), "x_scale must have shape ", shape_text(shape), ", got ", shape_text(xs.sizes()));
    TORCH_CHECK(ws.dim() == 2 && ws.size(0) == blocks_of(n) && ws.size(1) == blocks, "weight_scale must have shape (", blocks_of(n), ", ", blocks, "), got ",
                shape_text(ws.sizes()));
    TORCH_CHECK(!bias.defined() || (bias.dim() == 1 && bias.size(0) == n), "bias must have shape (", n, ",), got ", shape_text(bias.sizes()));
    for (const Tensor *t : {&xs, &w, &ws, &bias, &residual}) TORCH_CHECK(!t->defined() || t->device() == x.device(), "all tensors must be on the same device");
    for (const Tensor *t : {&bias, &residual})
        TORCH_CHECK(!t->defined() || t->scalar_type() == dtype, "bias and residual must have the result's type, ", dtype, ", got ", t->dtype());
    no_gradients("linear_fp8", {&x, &xs, &w, &ws, &bias, &residual});
    shape.back() = n;
    Tensor y;
    {
        const Released released;
        if (residual.defined()) residual = expanded(residual, shape);
        y = at::empty(shape, x.options().dtype(dtype));
        if (y.numel()) {
            const c10::DeviceGuard guard(x.device());
            // (rows that the entry point finds too far apart, as the last tokens of long sequences are, are copied)
            const auto near = [k](Rows t) { return t.stride < ADDER_CODES_STRIDE_MAX ? t : Rows{t.t.contiguous(), (long)k, t.rows}; };
            const Rows a = near(as_rows(x, k)), b = near(as_rows(w, k)), r = residual.defined() ? as_rows(residual, n) : Rows{Tensor(), 0, 0};
            xs = xs.contiguous();
            ws = ws.contiguous();
            if (bias.defined()) bias = bias.contiguous();
            const auto aligned = [](const Rows &t) { return !((reinterpret_cast<uintptr_t>(t.t.data_ptr()) | (uintptr_t)t.stride) & 15); };
            size_t need = 0;
            check(lib.codes_bytes(a.rows, (int)k, (int)n, type, aligned(a), aligned(b), &need), "adder_linear_codes_workspace_bytes");
            const Tensor space = bytes_for(need, x);
            check(lib.codes(static_cast<const unsigned char *>(a.t.data_ptr()), a.stride, xs.data_ptr<float>(), static_cast<const unsigned char *>(b.t.data_ptr()),
                            b.stride, ws.data_ptr<float>(), ptr(bias), ptr(r.t), r.stride, y.data_ptr(), act, a.rows, (int)k, (int)n, type, ptr(space), need,
                            stream_of(x)),
                  "adder_linear_codes");
        }
    }
    return THPVariable_Wrap(std::move(y));
    END_HANDLE_TH_ERRORS
}

// ---- gated linear layer -----------------------------------------------------------------------------------------------------
Tensor gated_forward(const Tensor &x, const Tensor &w, const Tensor &bias, int64_t act, Tensor *pre) {
    const int64_t n = w.size(0) / 2, k = w.size(1);
    c10::SmallVector<int64_t, 6> shape(x.sizes().begin(), x.sizes().end());
    shape.back() = n;
    Tensor y = at::empty(shape, x.options());
    if (pre) *pre = at::empty({x.numel() / k, 2 * n}, x.options());
    if (y.numel() == 0) return y;
    const c10::DeviceGuard guard(x.device());
    const Rows a = as_rows(x, k);
    size_t need = 0;
    const int type = type_of(x);
    check(lib.gated_fwd_bytes(a.rows, (int)k, (int)n, type, &need), "adder_gated_fwd_workspace_bytes");
    const Tensor ws = bytes_for(need, x);
    check(lib.gated_fwd(a.t.data_ptr(), a.stride, w.data_ptr(), ptr(bias), y.data_ptr(), pre ? pre->data_ptr() : nullptr, (int)act, a.rows, (int)k, (int)n, type,
                        ptr(ws), need, stream_of(x)),
          "adder_gated_fwd");
    return y;
}

struct GatedLinear : public torch::autograd::Function<GatedLinear> {
    static Variable forward(AutogradContext *ctx, const Variable &x, const Variable &w, const Maybe &has_bias, int64_t act) {
        const Tensor bias = has_bias.value_or(Tensor());
        const bool wx = x.requires_grad(), ww = w.requires_grad();
        Tensor pre;
        const Tensor y = gated_forward(x, w, bias, act, &pre);
        ctx->save_for_backward({ww ? x : Variable(), wx ? w : Variable(), pre});
        ctx->saved_data["act"] = act;
        ctx->saved_data["x"] = x.sizes().vec();
        ctx->saved_data["n"] = w.size(0) / 2;
        ctx->saved_data["bias"] = bias.defined();
        return y;
    }
    static variable_list backward(AutogradContext *ctx, const variable_list &grads) {
        refuse_in_capture("gated_linear");
        const auto saved = ctx->get_saved_variables();
        const Tensor &dy = grads[0];
        const bool want_x = ctx->needs_input_grad(0), want_w = ctx->needs_input_grad(1), want_b = ctx->saved_data["bias"].toBool() && ctx->needs_input_grad(2);
        variable_list out(4);
        if (!dy.defined()) return out;
        if (want_x || want_w || want_b) {
            const at::AutoGradMode off(false);
            const int64_t act = ctx->saved_data["act"].toInt(), n = ctx->saved_data["n"].toInt();
            const std::vector<int64_t> x_shape = ctx->saved_data["x"].toIntVector();
            const int64_t k = x_shape.back();
            const bool none = dy.numel() == 0;
            if (want_x) out[0] = filled(none, x_shape, dy.options());
            if (want_w) out[1] = filled(none, {2 * n, k}, dy.options());
            if (want_b) out[2] = filled(none, {2 * n}, dy.options());
            if (!none) {
                const c10::DeviceGuard guard(dy.device());
                const Rows d = as_rows(dy, n), x = want_w ? as_rows(saved[0], k) : Rows{Tensor(), (long)k, 0};
                size_t need = 0;
                const int type = type_of(dy);
                check(lib.gated_bwd_bytes(d.rows, (int)k, (int)n, type, &need), "adder_gated_bwd_workspace_bytes");
                const Tensor ws = bytes_for(need, dy);
                check(lib.gated_bwd(d.t.data_ptr(), d.stride, saved[2].data_ptr(), ptr(x.t), x.stride, ptr(saved[1]), ptr(out[0]), ptr(out[1]), ptr(out[2]),
                                    (int)act, d.rows, (int)k, (int)n, type, ptr(ws), need, stream_of(dy)),
                      "adder_gated_bwd");
            }
        }
        return once(std::move(out), "gated_linear");
    }
};

// gated_linear(x, weight, bias or None, act): plain GPU tensors, x float32 or bfloat16, no empty weight
PyObject *py_gated_linear(PyObject *, PyObject *const *args, Py_ssize_t count) {
    HANDLE_TH_ERRORS
    TORCH_CHECK(count == 4, "gated_linear: four arguments");
    const Tensor x = optional_tensor(args[0], "x");
    Tensor w = optional_tensor(args[1], "weight"), bias = optional_tensor(args[2], "bias");
    const int64_t act = integer(args[3]);
    TORCH_CHECK(w.dim() == 2 && w.size(0) % 2 == 0, "weight must have two dimensions, the first of two halves, got ", shape_text(w.sizes()));
    const int64_t n = w.size(0), k = w.size(1);
    TORCH_CHECK(x.dim() > 0 && x.size(-1) == k, "x has shape ", shape_text(x.sizes()), " but the weight expects ", k, " features");
    TORCH_CHECK(!bias.defined() || (bias.dim() == 1 && bias.size(0) == n), "bias must have shape (", n, ",), got ", shape_text(bias.sizes()));
    for (const Tensor *t : {&w, &bias}) {
        if (!t->defined()) continue;
        TORCH_CHECK(t->device() == x.device(), "all tensors must be on the same device");
        TORCH_CHECK(t->scalar_type() == x.scalar_type(), "all tensors must have the type of x, ", x.dtype(), ", got ", t->dtype());
    }
    Tensor y;
    {
        const Released released;
        w = w.contiguous();
        if (bias.defined()) bias = bias.contiguous();
        const bool grad = at::GradMode::is_enabled() && (wants_grad(x) || wants_grad(w) || wants_grad(bias));
        y = grad ? GatedLinear::apply(x, w, maybe(bias), act) : gated_forward(x, w, bias, act, nullptr);
    }
    return THPVariable_Wrap(std::move(y));
    END_HANDLE_TH_ERRORS
}

// ---- loss against a teacher's logits -------------------------------------------------------------------------------------------
struct Teacher {
    Tensor top, classes, labels;   // dense
    float temperature, alpha;
    int64_t ignore;
};
Tensor distill_forward(const Tensor &logits, const Teacher &t, Tensor *stats_out, Tensor *grad) {
    const c10::DeviceGuard guard(logits.device());
    const Rows l = as_rows(logits, logits.size(1));
    const int type = type_of(logits), classes = (int)logits.size(1);
    const auto floats = logits.options().dtype(at::kFloat);
    Tensor loss = at::empty({}, floats), stats = at::empty({(l.rows + 1) * ADDER_DISTILL_STATS}, floats);
    if (grad && lib.distill_in_rows(l.rows, classes, type)) *grad = at::empty(logits.sizes(), logits.options());
    size_t need = 0;
    check(lib.distill_bytes(l.rows, classes, type, &need), "adder_distill_workspace_bytes");
    const Tensor ws = bytes_for(need, logits);
    check(lib.distill_fwd(l.t.data_ptr(), l.stride, t.top.data_ptr(), reinterpret_cast<const long long *>(t.classes.data_ptr()),
                          reinterpret_cast<const long long *>(ptr(t.labels)), loss.data_ptr<float>(), stats.data_ptr<float>(), grad ? ptr(*grad) : nullptr,
                          t.temperature, t.alpha, t.ignore, l.rows, classes, (int)t.top.size(1), type, type_of(t.top), ptr(ws), need, stream_of(logits)),
          "adder_distill_fwd");
    if (stats_out) *stats_out = stats;
    return loss;
}

// The capture that the current stream is in; zero: none
int64_t capture_here() {
    const auto now = c10::hip::getCurrentHIPStream();
    if (now.id() == c10::hip::getDefaultHIPStream(now.device_index()).id()) return 0;   // (captures nothing, and must not be asked while another does)
    hipStreamCaptureStatus status = hipStreamCaptureStatusNone;
    unsigned long long id = 0;
    C10_HIP_CHECK(hipStreamGetCaptureInfo(now.stream(), &status, &id));
    return status == hipStreamCaptureStatusActive ? (int64_t)id : 0;
}

struct Distill : public torch::autograd::Function<Distill> {
    static Variable forward(AutogradContext *ctx, const Variable &logits, const Tensor &top, const Tensor &classes, const Maybe &labels, double temperature, double alpha,
                            int64_t ignore) {
        Tensor stats, grad;
        const Tensor loss = distill_forward(logits, {top, classes, labels.value_or(Tensor()), (float)temperature, (float)alpha, ignore}, &stats, &grad);
        ctx->save_for_backward({logits, top, classes, labels.value_or(Tensor()), stats});
        if (grad.defined()) {   // for a loss whose gradient is one
            const c10::DeviceGuard guard(logits.device());
            ctx->saved_data["grad"] = grad;
            ctx->saved_data["capture"] = capture_here();
        }
        ctx->saved_data["temperature"] = temperature;
        ctx->saved_data["alpha"] = alpha;
        ctx->saved_data["ignore"] = ignore;
        return loss;
    }
    static variable_list backward(AutogradContext *ctx, const variable_list &grads) {
        refuse_in_capture("distillation_loss");
        const auto saved = ctx->get_saved_variables();
        const Tensor &logits = saved[0], &top = saved[1];
        variable_list out(7);
        if (!grads[0].defined() || !ctx->needs_input_grad(0)) return out;
        {
            const at::AutoGradMode off(false);
            const c10::DeviceGuard guard(logits.device());
            // The forward's gradient is handed on, so a second pass over the same graph computes its own; so does one that is replayed without that forward, or
            // is not replayed with it: what was handed on would hold what the last replay, or its reader, left there.
            const auto ready = ctx->saved_data.find("grad");
            const bool unit = ready != ctx->saved_data.end() && ctx->saved_data["capture"].toInt() == capture_here();
            if (unit) {
                out[0] = ready->second.toTensor();
                ctx->saved_data.erase(ready);
            } else {
                out[0] = at::empty(logits.sizes(), logits.options());
            }
            const Rows l = as_rows(logits, logits.size(1));
            const Tensor up = grads[0].to(at::kFloat).contiguous();
            check(lib.distill_bwd(l.t.data_ptr(), l.stride, top.data_ptr(), reinterpret_cast<const long long *>(saved[2].data_ptr()),
                                  reinterpret_cast<const long long *>(ptr(saved[3])), saved[4].data_ptr<float>(), up.data_ptr<float>(), unit, out[0].data_ptr(),
                                  (float)ctx->saved_data["temperature"].toDouble(), (float)ctx->saved_data["alpha"].toDouble(), ctx->saved_data["ignore"].toInt(),
                                  l.rows, (int)logits.size(1), (int)top.size(1), type_of(logits), type_of(top), stream_of(logits)),
                  "adder_distill_bwd");
        }
        return once(std::move(out), "distillation_loss");
    }
};

// distillation_loss(logits, top_logits, top_classes, labels or None, temperature, alpha, ignore): plain GPU tensors, types and shapes looked at in distill.py
PyObject *py_distillation_loss(PyObject *, PyObject *const *args, Py_ssize_t count) {
    HANDLE_TH_ERRORS
    TORCH_CHECK(count == 7, "distillation_loss: seven arguments");
    const Tensor logits = optional_tensor(args[0], "logits");
    Teacher t{optional_tensor(args[1], "top_logits"), optional_tensor(args[2], "top_classes"), optional_tensor(args[3], "labels"), 0.f, 0.f, integer(args[6])};
    const double temperature = number(args[4]), alpha = number(args[5]);
    t.temperature = (float)temperature;
    t.alpha = (float)alpha;
    Tensor loss;
    {
        const Released released;
        t.top = t.top.detach().contiguous();
        t.classes = t.classes.contiguous();
        if (t.labels.defined()) t.labels = t.labels.contiguous();
        loss = at::GradMode::is_enabled() && logits.requires_grad() ? Distill::apply(logits, t.top, t.classes, maybe(t.labels), temperature, alpha, t.ignore)
                                                                     : distill_forward(logits, t, nullptr, nullptr);
    }
    return THPVariable_Wrap(std::move(loss));
    END_HANDLE_TH_ERRORS
}

PyMethodDef method(const char *name, PyObject *(*of)(PyObject *, PyObject *const *, Py_ssize_t)) {
    return {name, reinterpret_cast<PyCFunction>(reinterpret_cast<void *>(of)), METH_FASTCALL, nullptr};
}

}  // namespace

const std::vector<PyMethodDef> block_methods = {
    method("rms_norm", py_rms_norm),       method("rms_norm_fp8", py_rms_norm_fp8), method("quantize", py_quantize),
    method("quantize_weight", py_quantize_weight), method("linear_fp8", py_linear_fp8),     method("gated_linear", py_gated_linear),
    method("distillation_loss", py_distillation_loss),
};

}  // namespace nodes
