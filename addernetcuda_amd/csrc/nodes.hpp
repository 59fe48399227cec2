// What the files of the host module share: the library's entry points, and how tensors reach them.
#pragma once
#include <Python.h>

#include <ATen/ops/empty.h>
#include <ATen/ops/zeros.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPGraphsC10Utils.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/accumulate_grad.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/graph_task.h>
#include <torch/csrc/autograd/python_variable.h>

#include <string>
#include <unordered_set>
#include <vector>

#include "../../include/addernet_hip.h"

namespace nodes {

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
    decltype(&adder_rms_norm_fwd) rms_fwd;
    decltype(&adder_rms_norm_fwd_codes) rms_fwd_codes;
    decltype(&adder_rms_norm_bwd_workspace_bytes) rms_bwd_bytes;
    decltype(&adder_rms_norm_bwd) rms_bwd;
    decltype(&adder_quantize) quantize;
    decltype(&adder_quantize_weight) quantize_weight;
    decltype(&adder_linear_codes_workspace_bytes) codes_bytes;
    decltype(&adder_linear_codes) codes;
    decltype(&adder_gated_fwd_workspace_bytes) gated_fwd_bytes;
    decltype(&adder_gated_fwd) gated_fwd;
    decltype(&adder_gated_bwd_workspace_bytes) gated_bwd_bytes;
    decltype(&adder_gated_bwd) gated_bwd;
    decltype(&adder_distill_in_rows) distill_in_rows;
    decltype(&adder_distill_workspace_bytes) distill_bytes;
    decltype(&adder_distill_fwd) distill_fwd;
    decltype(&adder_distill_bwd) distill_bwd;
};
extern Library lib;

inline void check(int status, const char *what) {
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

inline int type_of(const Tensor &t) { return t.scalar_type() == at::kBFloat16 ? ADDER_TYPE_BF16 : ADDER_TYPE_F32; }
inline void *stream_of(const Tensor &t) { return c10::hip::getCurrentHIPStream(t.device().index()).stream(); }
inline void *ptr(const Tensor &t) { return t.defined() ? t.data_ptr() : nullptr; }
inline Tensor bytes_for(size_t n, const Tensor &like) {
    return n ? at::empty({(int64_t)n}, like.options().dtype(at::kByte)) : Tensor();
}
inline Tensor filled(bool zeros, at::IntArrayRef shape, const at::TensorOptions &options) {
    return zeros ? at::zeros(shape, options) : at::empty(shape, options);
}
inline std::string shape_text(at::IntArrayRef s) {   // as Python prints it
    std::string t = "(";
    for (size_t i = 0; i < s.size(); ++i) t += std::to_string(s[i]) + (i + 1 < s.size() ? ", " : s.size() == 1 ? "," : "");
    return t + ")";
}

// t as rows of `width` neighbouring values, and their stride: a view where it is one.  Values of one row lie side by side, and rows that are not all
// the same one do not overlap.
struct Rows { Tensor t; long stride, rows; };
inline Rows as_rows(const Tensor &t, int64_t width) {
    const int64_t rows = t.numel() / width;
    if (t.is_contiguous()) return {t, (long)width, (long)rows};
    Tensor v = t.dim() == 2 && t.size(1) == width ? t : t.reshape({rows, width});   // (two dimensions may also be one row: all of them normalised)
    if ((width > 1 && v.stride(1) != 1) || (rows > 1 && v.stride(0) < width && v.stride(0) != 0)) v = v.contiguous();
    return {v, rows > 1 ? (long)v.stride(0) : (long)width, (long)rows};
}

// Calls f with the leaves' nodes that a backward pass reaches from `from` on (inside a pass: this one), each once, until it says true
template <class F>
bool any_leaf(torch::autograd::Node *from, const F &f) {
    const auto *runs = torch::autograd::get_current_graph_task_exec_info();   // of a pass for some inputs only: what it runs
    std::vector<torch::autograd::Node *> open{from};
    std::unordered_set<torch::autograd::Node *> seen{from};
    while (!open.empty()) {
        torch::autograd::Node *node = open.back();
        open.pop_back();
        if (auto *leaf = dynamic_cast<torch::autograd::AccumulateGrad *>(node))
            if (f(*leaf)) return true;
        for (const auto &edge : node->next_edges()) {
            torch::autograd::Node *next = edge.function.get();
            if (!next || !seen.insert(next).second) continue;
            if (runs && !runs->empty()) {
                const auto it = runs->find(next);
                if (it == runs->end() || !it->second.should_execute()) continue;
            }
            open.push_back(next);
        }
    }
    return false;
}

// A leaf whose earlier graph still lives keeps the stream that its gradients are added on.  Where that is the default stream, a gradient that is captured on
// another one would have it wait for the capture, which no capture allows and which ends the process: said here instead, before anything is captured for it.
// All leaves that the pass comes to behind this node are looked at, whatever lies between (a cast, a view, other layers): the first of these nodes speaks for them.
inline void refuse_in_capture(const char *what) {
    const auto node = torch::autograd::get_current_node();
    if (!node) return;
    const auto now = c10::hip::getCurrentHIPStream();
    if (now.id() == c10::hip::getDefaultHIPStream(now.device_index()).id()) return;   // (captures nothing)
    if (c10::hip::currentStreamCaptureStatusMayInitCtx() == c10::hip::CaptureStatus::None) return;
    const bool waits = any_leaf(node.get(), [](torch::autograd::AccumulateGrad &leaf) {
        const auto of = leaf.stream();
        return of && of->device_type() == c10::kCUDA && of->id() == c10::hip::getDefaultHIPStream(of->device_index()).id();
    });
    TORCH_CHECK(!waits, what,
                ": a backward pass cannot be captured while a graph of the same leaves that was made on the default stream lives; drop its tensors first, or make it "
                "on the stream of the capture");
}

// Gradients that these nodes give have no formula to be differentiated again: whoever tries is told so
inline variable_list once(variable_list grads, const char *what) {
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

// Arguments that may be absent reach a node as optionals; its edges count those that are there
typedef std::optional<Variable> Maybe;
inline Maybe maybe(const Tensor &t) { return t.defined() ? Maybe(t) : Maybe(); }

inline Tensor optional_tensor(PyObject *o, const char *name) {
    if (o == Py_None) return Tensor();
    if (!THPVariable_Check(o)) throw torch::TypeError(std::string(name) + " must be a torch.Tensor");
    return THPVariable_Unpack(o);
}

extern const std::vector<PyMethodDef> block_methods;   // (nodes_blocks.cpp)

}  // namespace nodes
