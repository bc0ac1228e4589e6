// What the host sides of the operators around the attention share: rows as the kernels read them, their autograd nodes, checks of arguments.
#pragma once
#include "block.h"

#include <c10/hip/HIPGraphsC10Utils.h>

namespace {

using namespace llsa_host;

inline int64_t pad8(int64_t n) { return (n + 7) / 8 * 8; }
inline bool aligned(const Tensor& t) { return reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0; }
inline std::string name_of(at::ScalarType t) { return "torch." + std::string(torch::getTHPDtype(t)->name); }

inline int dtype_of(const Tensor& t, bool f32_too, const char* what) {
    switch (t.scalar_type()) {
        case at::kBFloat16: return LLSA_DTYPE_BF16;
        case at::kHalf: return LLSA_DTYPE_F16;
        case at::kFloat:
            if (f32_too) return LLSA_DTYPE_F32;
            break;
        default: break;
    }
    fail(Failure::kNotImplemented, std::string(what) + (f32_too ? " takes bf16, fp16 or fp32 (got " : " takes bf16 or fp16 (got ") + name_of(t.scalar_type()) + ")");
}

// A tensor of rows along its last dimension: the rows one step apart, elements next to each other.  A copy where it is laid out otherwise.
struct Rows {
    Tensor t;
    int64_t ld = 0, count = 0, cols = 0;
    void* p() const { return t.defined() ? t.data_ptr() : nullptr; }
};
// What the memory of a tensor has to hold for the kernels: its values, not those of a view that torch negates on reading
inline Tensor in_memory(const Tensor& t) { return t.is_neg() ? t.resolve_neg() : t; }
inline Rows rows_of(const Tensor& given) {
    const Tensor t = in_memory(given);
    Rows r;
    r.cols = t.size(-1);
    r.count = r.cols > 0 ? t.numel() / r.cols : 0;
    bool fits = t.stride(-1) == 1 || r.cols == 1;
    int64_t step = 0, span = 0;                               // of the innermost leading dimension, and what the ones seen so far step over
    for (int64_t i = t.dim() - 2; i >= 0; i--) {
        if (t.size(i) == 1) continue;
        if (step == 0) {
            step = t.stride(i);
            fits = fits && step >= r.cols;
            span = step * t.size(i);
        } else {
            fits = fits && t.stride(i) == span;
            span *= t.size(i);
        }
    }
    r.t = fits ? t : t.contiguous();
    r.ld = fits && step != 0 ? step : r.cols;
    return r;
}

class Call {
public:
    Call(const Library& lib, const Tensor& on) : lib_(lib), stream_(lib.stream(on)), options_(on.options()) {}
    const Library& lib() const { return lib_; }
    void* stream() const { return stream_; }
    Tensor rows(int64_t count, int64_t cols) const { return at::empty({count, pad8(cols)}, options_); }
    Tensor bytes(int64_t n) const { return n > 0 ? at::empty({n}, options_.dtype(at::kByte)) : Tensor(); }
    // Rows that the products read: 16-byte aligned, whole pieces of eight elements.  Matrices that are not are copied, in one launch.
    void operands(std::initializer_list<std::pair<const Tensor*, Rows*>> all) const {
        llsa_pad_job jobs[LLSA_PAD_JOBS];
        int n = 0;
        for (const auto& [t, r] : all) {
            *r = rows_of(*t);
            if (aligned(r->t) && r->ld % 8 == 0 && r->cols % 8 == 0 && r->ld <= (int64_t(1) << 23)) continue;
            const Tensor y = rows(r->count, r->cols);
            jobs[n++] = llsa_pad_job{r->p(), y.data_ptr(), r->ld, y.size(1), r->count, static_cast<int32_t>(r->cols), 0};
            copied_.push_back(r->t);                          // (until the copies are issued)
            r->t = y;
            r->ld = y.size(1);
        }
        if (n > 0) lib_.check(lib_.pad_rows(jobs, n, stream_), "pad_rows");
        copied_.clear();
    }
    // Rows of a residual, which are read as they lie, up to 2^23 elements apart
    Rows addend(const Tensor* t) const {
        Rows r;
        if (t == nullptr) return r;
        r = rows_of(*t);
        if (r.ld > (int64_t(1) << 23)) {
            r.t = r.t.contiguous();
            r.ld = r.cols;
        }
        return r;
    }
    Rows operand(const Tensor& t) const {
        Rows r;
        operands({{&t, &r}});
        return r;
    }

private:
    const Library& lib_;
    void* stream_;
    at::TensorOptions options_;
    mutable std::vector<Tensor> copied_;
};

// The node of an operator with one output: what is common to the three of them.  `kept` are the saved tensors in the order run() unpacks them.
struct BlockNode : public Node {
    struct Kind {                         // of a saved tensor, which its hooks have to give back: the kernels' sizes come from the node.  Strides may differ.
        bool defined;
        std::vector<int64_t> sizes;
        at::ScalarType type;
        at::Device device;
    };
    std::shared_ptr<Library> lib;
    std::vector<SavedVariable> kept;
    std::vector<Kind> kinds;
    bool released = false;

    void release_variables() override {
        std::lock_guard<std::mutex> lock(mutex_);
        released = true;
        for (SavedVariable& s : kept) s.reset_data();
    }
    variable_list apply(variable_list&& grads) override {
        std::lock_guard<std::mutex> lock(mutex_);
        return in_engine([&]() -> variable_list {
            if (released) fail(Failure::kRuntime, torch::autograd::ERR_BACKWARD_TWICE);
            if (at::GradMode::is_enabled()) fail(Failure::kNotImplemented, "llsa_amd " + name() + " has no second derivative (create_graph=True)");
            if (!grads[0].defined()) return variable_list(num_outputs());
            // (before the autograd keys are left out: a hook may run the forward again)
            std::vector<Tensor> saved;
            for (size_t i = 0; i < kept.size(); i++) {
                saved.push_back(kept[i].unpack(shared_from_this()));
                const Tensor& t = saved.back();
                const Kind& k = kinds[i];
                if (t.defined() != k.defined || (k.defined && (t.layout() != at::kStrided || t.sizes() != k.sizes || t.scalar_type() != k.type || t.device() != k.device)))
                    fail(Failure::kRuntime, "llsa_amd: a saved-tensor hook returned another tensor than it was given");
            }
            at::AutoDispatchBelowADInplaceOrView below;
            c10::OptionalDeviceGuard guard(lib->device ? std::optional<at::Device>(grads[0].device()) : std::nullopt);
            return run(grads[0], saved);
        });
    }
    virtual variable_list run(const Tensor& grad, const std::vector<Tensor>& saved) = 0;
    // a tensor that only the kernels read, as they left it
    static Tensor as_kept(const Tensor& t) { return t.is_contiguous() && aligned(t) && !t.is_neg() ? t : t.clone(at::MemoryFormat::Contiguous).resolve_neg(); }
    void keep(const Tensor& t, const Tensor& input) {
        kinds.push_back(t.defined() ? Kind{true, t.sizes().vec(), t.scalar_type(), t.device()} : Kind{false, {}, at::kFloat, at::kCPU});
        kept.emplace_back(t.is_same(input) ? input : t, false);
    }
};

// A graph that is being captured must not reach gradients that another graph on another stream holds: a leaf has one accumulator, tied to the stream
// it was made on, and a captured backward that has to wait for that stream ends the process (of any operator).
inline void refuse_foreign_accumulators(const Library& lib, std::initializer_list<const Tensor*> all) {
    if (!lib.device || !at::GradMode::is_enabled()) return;
    if (c10::hip::currentStreamCaptureStatusMayInitCtx() == c10::hip::CaptureStatus::None) return;
    for (const Tensor* t : all) {
        if (t == nullptr || !t->requires_grad() || !t->is_leaf() || !t->is_cuda()) continue;
        const auto accumulator = torch::autograd::impl::try_get_grad_accumulator(*t);
        if (!accumulator) continue;
        const std::optional<c10::Stream> made_on = accumulator->stream();
        const c10::Stream now = c10::hip::getCurrentHIPStream(t->device().index()).unwrap();
        // (number and device alone: autograd's streams call their devices CUDA, these call them HIP, and so no two of them are equal)
        if (made_on.has_value() && (made_on->id() != now.id() || made_on->device_index() != now.device_index()))
            fail(Failure::kRuntime, "llsa_amd: a graph is being captured, and an input's gradient belongs to another graph that is still alive: let go of it first "
                                    "(delete the outputs of earlier forward passes)");
    }
}

// the checks all three begin with
inline void begin(const Library& lib, const char* what, const Tensor& x, std::initializer_list<const Tensor*> all) {
    if (torch::jit::tracer::isTracing()) fail(Failure::kRuntime, std::string("llsa_amd ") + what + " cannot be recorded by torch.jit.trace");
    refuse_transforms(all);
    for (const Tensor* t : all) {
        if (t == nullptr) continue;
        if (t->layout() != at::kStrided) fail(Failure::kNotImplemented, std::string(what) + " takes dense tensors");
        if (t->device() != x.device()) fail(Failure::kValue, std::string(what) + ": all tensors must be on one device");
    }
    lib.on_device(x);
    refuse_foreign_accumulators(lib, all);
}
inline bool wants(std::initializer_list<const Tensor*> all) {
    if (!at::GradMode::is_enabled()) return false;
    for (const Tensor* t : all)
        if (t != nullptr && t->requires_grad()) return true;
    return false;
}
template <typename N>
std::shared_ptr<N> make_node(const std::shared_ptr<Library>& lib) {
    auto node = std::shared_ptr<N>(new N, torch::autograd::deleteNode);
    node->lib = lib;
    return node;
}
inline variable_list present(std::initializer_list<const Tensor*> all) {
    variable_list v;
    for (const Tensor* t : all)
        if (t != nullptr) v.push_back(*t);
    return v;
}

inline void check_vector(const char* what, const char* name, const Tensor* t, at::IntArrayRef sizes) {
    if (t != nullptr && t->sizes() != sizes)
        fail(Failure::kValue, std::string(what) + ": " + name + " must be " + text_of(sizes) + " (got " + text_of(t->sizes()) + ")");
}
// samples: the first dimension, where there is one beside the channels
inline int64_t samples_of(const char* what, const char* name, const Tensor& x) {
    if (x.dim() < 2) fail(Failure::kValue, std::string(what) + ": " + name + " needs a dimension of samples in front of the channels");
    return x.size(0);
}

// The arguments that linear and feed_forward share
struct LayerInputs {
    const Tensor *x, *gate, *residual;
    int64_t rows, samples;
    int64_t per_sample() const { return std::max<int64_t>(1, samples > 0 ? rows / samples : rows); }
};
inline LayerInputs layer_inputs(const char* what, const Tensor& x, const Tensor* gate, const Tensor* residual, int64_t out) {
    LayerInputs i{&x, gate, residual, 1, 1};
    for (int64_t d = 0; d + 1 < x.dim(); d++) i.rows *= x.size(d);
    if (gate != nullptr) {
        i.samples = samples_of(what, "gate", x);
        check_vector(what, "gate", gate, {i.samples, out});
    }
    std::vector<int64_t> sizes = x.sizes().vec();
    sizes.back() = out;
    check_vector(what, "residual", residual, sizes);
    if (i.rows >= (int64_t(1) << 31) - (1 << 16)) fail(Failure::kValue, std::string(what) + ": too many rows (" + std::to_string(i.rows) + ")");
    return i;
}
inline void check_weight(const char* what, const char* name, const Tensor& w, int64_t in, const Tensor& x) {
    if (w.dim() != 2 || w.size(0) < 1 || w.size(1) < 1 || (in >= 0 && w.size(1) != in))
        fail(Failure::kValue, std::string(what) + ": " + name + " must be (channels out, " + (in >= 0 ? std::to_string(in) : std::string("channels in")) + ") (got " + text_of(w.sizes()) + ")");
    if (w.size(0) >= (1 << 23) || w.size(1) >= (1 << 23)) fail(Failure::kValue, std::string(what) + ": too many channels");
}
inline void same_types(const char* what, const Tensor& x, std::initializer_list<const Tensor*> all) {
    for (const Tensor* t : all)
        if (t != nullptr && t->scalar_type() != x.scalar_type())
            fail(Failure::kValue, std::string(what) + ": all tensors must have x's dtype, " + name_of(x.scalar_type()) + " (got " + name_of(t->scalar_type()) + ")");
}
inline Tensor dense_vector(const Tensor* t) {                        // (N) or (samples, N) with elements next to each other
    if (t == nullptr) return Tensor();
    const Tensor v = in_memory(*t);
    return v.size(-1) <= 1 || v.stride(-1) == 1 ? v : v.contiguous();
}
inline int activation(const char* what, int64_t act) {
    if (act < LLSA_ACT_NONE || act > LLSA_ACT_GELU_TANH) fail(Failure::kValue, std::string(what) + ": unknown activation");
    return static_cast<int>(act);
}
inline Tensor zeros_like_weight(int64_t n, int64_t k, const Tensor& like) { return at::zeros({n, k}, like.options()); }

// An operand of the forward, which may be a copy with padded rows, of which `cols` elements count
inline Rows kept_operand(const Call& call, const Tensor& t, int64_t cols) {
    Rows r = call.operand(t);
    r.cols = cols;
    return r;
}

}  // namespace
