// What the translation units of the host module share: errors, the library's entry points, checks of tensors.
#pragma once
#include <torch/csrc/Dtype.h>
#include <torch/csrc/DynamicTypes.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/function.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/saved_variable.h>
#include <torch/csrc/autograd/variable.h>
#include <torch/csrc/jit/frontend/tracer.h>
#include <torch/csrc/utils/pybind.h>
#include <torch/extension.h>
#include <c10/hip/HIPStream.h>
#include <hip/hip_runtime_api.h>

#include <algorithm>
#include <array>
#include <mutex>
#include <optional>
#include <string>
#include <utility>
#include <vector>

#include "../../../include/llsa_hip.h"

namespace llsa_host {

namespace py = pybind11;
using at::Tensor;
using torch::autograd::Node;
using torch::autograd::SavedVariable;
using torch::autograd::variable_list;

// ---------------------------------------------------------------------------------------
// errors: which Python exception, and its text
// ---------------------------------------------------------------------------------------
struct Failure {
    enum Kind { kValue, kNotImplemented, kRuntime, kLibrary } kind;
    std::string text;
};
inline PyObject* g_library_error = nullptr;      // llsa_amd._lib.LlsaError

[[noreturn]] inline void fail(Failure::Kind kind, std::string text) { throw Failure{kind, std::move(text)}; }

inline void set_python_error(const Failure& f) {                 // with the interpreter lock held
    PyObject* type = f.kind == Failure::kValue            ? PyExc_ValueError
                     : f.kind == Failure::kNotImplemented ? PyExc_NotImplementedError
                     : f.kind == Failure::kLibrary && g_library_error != nullptr ? g_library_error
                                                          : PyExc_RuntimeError;
    PyErr_SetString(type, f.text.c_str());
}

template <typename Fn>
auto without_interpreter(Fn fn) {
    std::optional<Failure> failure;
    {
        py::gil_scoped_release release;
        try {
            return fn();
        } catch (const Failure& f) {
            failure = f;
        }
    }
    set_python_error(*failure);
    throw py::error_already_set();
}
// the same on a thread of the autograd engine, which does not hold the lock
template <typename Fn>
auto in_engine(Fn fn) {
    try {
        return fn();
    } catch (const Failure& f) {
        py::gil_scoped_acquire acquire;
        set_python_error(f);
        python_error e;
        e.persist();
        throw e;
    }
}

// ---------------------------------------------------------------------------------------
// the library
// ---------------------------------------------------------------------------------------
struct Library {
    decltype(&llsa_last_error_string) last_error_string;
    decltype(&llsa_pool_pyramid_fwd) pool_pyramid_fwd;
    decltype(&llsa_topk_dense_tiles) topk_dense_tiles;
    decltype(&llsa_topk_sparse_tiles) topk_sparse_tiles;
    decltype(&llsa_topk_cascade_tiles) topk_cascade_tiles;
    decltype(&llsa_topk_cascade_max_parents) topk_cascade_max_parents;
    decltype(&llsa_attn_fwd) attn_fwd;
    decltype(&llsa_attn_fwd_lists) attn_fwd_lists;
    decltype(&llsa_attn_fwd_selects) attn_fwd_selects;
    decltype(&llsa_transpose_indices_multi) transpose_indices_multi;
    decltype(&llsa_transpose_one_launch) transpose_one_launch;
    decltype(&llsa_transpose_nested_bytes) transpose_nested_bytes;
    decltype(&llsa_work_list_len) work_list_len;
    decltype(&llsa_fine_chunk_for) fine_chunk_for;
    decltype(&llsa_attn_bwd_workspace_bytes) attn_bwd_workspace_bytes;
    decltype(&llsa_attn_bwd) attn_bwd;
    decltype(&llsa_gather_rows) gather_rows;
    decltype(&llsa_layer_norm_fwd) layer_norm_fwd;
    decltype(&llsa_layer_norm_bwd) layer_norm_bwd;
    decltype(&llsa_layer_norm_bwd_workspace_bytes) layer_norm_bwd_workspace_bytes;
    decltype(&llsa_linear_fwd) linear_fwd;
    decltype(&llsa_linear_dz) linear_dz;
    decltype(&llsa_linear_dx) linear_dx;
    decltype(&llsa_linear_dw) linear_dw;
    decltype(&llsa_linear_gate_rows) linear_gate_rows;
    decltype(&llsa_linear_dw_workspace_bytes) linear_dw_workspace_bytes;
    decltype(&llsa_linear_dz_workspace_bytes) linear_dz_workspace_bytes;
    decltype(&llsa_pad_rows) pad_rows;
    decltype(&llsa_quantize_rows) quantize_rows;
    decltype(&llsa_linear_int8) linear_int8;
    decltype(&llsa_route_tokens) route_tokens;
    decltype(&llsa_route_tokens_bwd) route_tokens_bwd;
    decltype(&llsa_route_workspace_bytes) route_workspace_bytes;
    decltype(&llsa_experts_gather) experts_gather;
    decltype(&llsa_experts_gathers) experts_gathers;
    decltype(&llsa_experts_fwd) experts_fwd;
    decltype(&llsa_experts_dx) experts_dx;
    decltype(&llsa_experts_dz) experts_dz;
    decltype(&llsa_experts_dw) experts_dw;
    decltype(&llsa_experts_dweights_workspace_bytes) experts_dweights_workspace_bytes;
    decltype(&llsa_experts_combine) experts_combine;
    decltype(&llsa_experts_dweights) experts_dweights;
    decltype(&llsa_experts_dw_workspace_bytes) experts_dw_workspace_bytes;
    bool device;                          // false: the CPU emulation build the tests install

    Library(const std::map<std::string, uintptr_t>& at_, bool device_) : device(device_) {
        auto get = [&](const char* name, auto& fn) { fn = reinterpret_cast<std::decay_t<decltype(fn)>>(at_.at(name)); };
        get("llsa_last_error_string", last_error_string);
        get("llsa_pool_pyramid_fwd", pool_pyramid_fwd);
        get("llsa_topk_dense_tiles", topk_dense_tiles);
        get("llsa_topk_sparse_tiles", topk_sparse_tiles);
        get("llsa_topk_cascade_tiles", topk_cascade_tiles);
        get("llsa_topk_cascade_max_parents", topk_cascade_max_parents);
        get("llsa_attn_fwd", attn_fwd);
        get("llsa_attn_fwd_lists", attn_fwd_lists);
        get("llsa_attn_fwd_selects", attn_fwd_selects);
        get("llsa_transpose_indices_multi", transpose_indices_multi);
        get("llsa_transpose_one_launch", transpose_one_launch);
        get("llsa_transpose_nested_bytes", transpose_nested_bytes);
        get("llsa_work_list_len", work_list_len);
        get("llsa_fine_chunk_for", fine_chunk_for);
        get("llsa_attn_bwd_workspace_bytes", attn_bwd_workspace_bytes);
        get("llsa_attn_bwd", attn_bwd);
        get("llsa_gather_rows", gather_rows);
        get("llsa_layer_norm_fwd", layer_norm_fwd);
        get("llsa_layer_norm_bwd", layer_norm_bwd);
        get("llsa_layer_norm_bwd_workspace_bytes", layer_norm_bwd_workspace_bytes);
        get("llsa_linear_fwd", linear_fwd);
        get("llsa_linear_dz", linear_dz);
        get("llsa_linear_dx", linear_dx);
        get("llsa_linear_dw", linear_dw);
        get("llsa_linear_gate_rows", linear_gate_rows);
        get("llsa_linear_dw_workspace_bytes", linear_dw_workspace_bytes);
        get("llsa_linear_dz_workspace_bytes", linear_dz_workspace_bytes);
        get("llsa_pad_rows", pad_rows);
        get("llsa_quantize_rows", quantize_rows);
        get("llsa_linear_int8", linear_int8);
        get("llsa_route_tokens", route_tokens);
        get("llsa_route_tokens_bwd", route_tokens_bwd);
        get("llsa_route_workspace_bytes", route_workspace_bytes);
        get("llsa_experts_gather", experts_gather);
        get("llsa_experts_gathers", experts_gathers);
        get("llsa_experts_fwd", experts_fwd);
        get("llsa_experts_dx", experts_dx);
        get("llsa_experts_dz", experts_dz);
        get("llsa_experts_dw", experts_dw);
        get("llsa_experts_dweights_workspace_bytes", experts_dweights_workspace_bytes);
        get("llsa_experts_combine", experts_combine);
        get("llsa_experts_dweights", experts_dweights);
        get("llsa_experts_dw_workspace_bytes", experts_dw_workspace_bytes);
    }
    void check(int rc, const char* what) const {
        if (rc != 0) fail(Failure::kLibrary, std::string(what) + " failed (" + std::to_string(rc) + "): " + last_error_string());
    }
    void on_device(const Tensor& t) const {
        if (device && !t.is_cuda())
            fail(Failure::kRuntime, "llsa_amd runs on an AMD GPU only (got a CPU tensor); there is no CPU implementation");
    }
    void* stream(const Tensor& t) const {
        return device ? static_cast<void*>(c10::hip::getCurrentHIPStream(t.device().index()).stream()) : nullptr;
    }
};

inline std::string text_of(at::IntArrayRef v) {
    std::string s = "(";
    for (size_t i = 0; i < v.size(); i++) s += (i ? ", " : "") + std::to_string(v[i]);
    return s + ")";
}

inline bool strides_multiple(at::IntArrayRef st, int64_t m) {
    for (size_t i = 0; i + 1 < st.size(); i++)
        if (st[i] % m != 0) return false;
    return true;
}
// Whether no two elements of such a tensor share memory (an expanded one's do): every dimension steps over all that the smaller steps span.
inline bool own_places(const std::array<int64_t, 4>& sizes, const std::array<int64_t, 4>& st) {
    std::array<std::pair<int64_t, int64_t>, 4> dims;          // step, entries
    for (int i = 0; i < 4; i++) dims[i] = {sizes[i] > 1 ? st[i] : 0, sizes[i]};
    std::sort(dims.begin(), dims.end());
    int64_t span = 1;
    for (const auto& [step, n] : dims) {
        if (n > 1 && step < span) return false;
        span += step * (n - 1);
    }
    return true;
}
// last stride 1 and every row 16-byte aligned: what the kernels' 16-byte loads need
inline bool rows_ok(const Tensor& t) {
    return t.stride(-1) == 1 && reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0 && strides_multiple(t.strides(), 8);
}
inline Tensor as_rows(const Tensor& t) { return rows_ok(t) ? t : t.contiguous(); }
// a tensor as the kernels need it, wherever and with whatever strides a caller or a saved-tensor hook has put it
inline Tensor restored(const Tensor& t, bool contiguous = false) {
    const bool usable = !t.defined() || (rows_ok(t) && (!contiguous || t.is_contiguous()));
    return usable ? t : t.clone(at::MemoryFormat::Contiguous);
}

inline int64_t align_up(int64_t n, int64_t a) { return (n + a - 1) / a * a; }

// What torch.autograd.Function refuses for the operators written in Python, an operator whose node is native has to refuse itself:
// inputs that carry a tangent (the kernels have no forward-mode rule; without this the result would carry none, which reads
// as a derivative of zero) and torch.func's transforms, whose tensors have no data.
inline void refuse_transforms(std::initializer_list<const Tensor*> inputs) {
    const c10::DispatchKeySet active = c10::impl::tls_local_dispatch_key_set().included_;
    if (active.has(c10::DispatchKey::FuncTorchDynamicLayerFrontMode) || active.has(c10::DispatchKey::FuncTorchDynamicLayerBackMode))
        fail(Failure::kRuntime, "llsa_amd operators do not work under functorch transforms (vmap, grad, jvp, jacrev, ...)");
    for (const Tensor* t : inputs)
        if (t != nullptr && t->_fw_grad(/*level=*/0).defined())
            fail(Failure::kNotImplemented, "llsa_amd operators have no jvp function: forward mode AD is not supported");
}
inline const Tensor* address(const std::optional<Tensor>& t) { return t.has_value() ? &*t : nullptr; }

}  // namespace llsa_host
