// The host side of the linear layer in 8-bit integers (quantize_rows, linear_int8): argument checks and the calls of the C ABI.  No gradients.
#include "block_common.h"

namespace {

int64_t pad16(int64_t n) { return (n + 15) / 16 * 16; }

void refuse_gradients(const char* what, std::initializer_list<const Tensor*> all) {
    if (wants(all))
        fail(Failure::kNotImplemented, std::string(what) + " has no gradient: call it under torch.no_grad(), or with tensors that want none");
}
// what the kernels write whole numbers of: all of x's sizes
std::vector<int64_t> without_last(const Tensor& x) { return std::vector<int64_t>(x.sizes().begin(), x.sizes().end() - 1); }

// rows of integers as the products read them (16-byte aligned, whole pieces of sixteen), or a copy job, out of what `copied` keeps until it is issued
Rows integers(const Tensor& given, llsa_quantize_args& a, std::vector<Tensor>& copied) {
    Rows r = rows_of(given);
    if (aligned(r.t) && r.ld % 16 == 0 && r.cols % 16 == 0 && r.ld <= (int64_t(1) << 23)) return r;
    Rows y;
    y.t = at::empty({r.count, pad16(r.cols)}, r.t.options());
    y.ld = y.t.size(1); y.count = r.count; y.cols = r.cols;
    copied.push_back(r.t);
    a.pad[a.pads++] = llsa_pad_job{r.p(), y.p(), r.ld, y.ld, r.count, static_cast<int32_t>(r.cols), 0};
    return y;
}
int64_t row_length(const char* what, const Tensor& x) {
    if (x.dim() < 1 || x.size(-1) < 1 || x.size(-1) >= (1 << 23)) fail(Failure::kValue, std::string(what) + ": x needs a dimension of channels (got " + text_of(x.sizes()) + ")");
    return x.size(-1);
}
int64_t row_count(const char* what, const Tensor& x) {
    int64_t rows = 1;
    for (int64_t d = 0; d + 1 < x.dim(); d++) rows *= x.size(d);
    if (rows >= (int64_t(1) << 31) - (1 << 16)) fail(Failure::kValue, std::string(what) + ": too many rows (" + std::to_string(rows) + ")");
    return rows;
}
// (`padded`: rows of q are a multiple of 16 long)
void quantize_job(llsa_quantize_args& a, const Rows& x, const Tensor& q, const Tensor& scale, int dtype, bool padded) {
    a.x = x.p(); a.ldx = x.ld; a.rows = x.count; a.K = static_cast<int32_t>(x.cols); a.dtype = dtype;
    a.q = q.data_ptr(); a.ldq = padded ? pad16(x.cols) : x.cols; a.padded = padded; a.scale = scale.data_ptr<float>();
}

std::pair<Tensor, Tensor> quantize_rows(const std::shared_ptr<Library>& lib, const Tensor& x_in) {
    const char* const what = "quantize_rows";
    begin(*lib, what, x_in, {&x_in});
    const int dtype = dtype_of(x_in, true, what);
    const int64_t K = row_length(what, x_in);
    const int64_t count = row_count(what, x_in);
    refuse_gradients(what, {&x_in});
    at::AutoDispatchBelowADInplaceOrView below;
    c10::OptionalDeviceGuard guard(lib->device ? std::optional<at::Device>(x_in.device()) : std::nullopt);
    const Tensor q = at::empty(x_in.sizes(), x_in.options().dtype(at::kChar)), scale = at::empty(without_last(x_in), x_in.options().dtype(at::kFloat));
    if (count > 0) {
        const Rows x = rows_of(x_in);
        llsa_quantize_args a{};
        quantize_job(a, x, q, scale, dtype, K % 16 == 0);
        lib->check(lib->quantize_rows(&a, lib->stream(x_in)), what);
    }
    return {q, scale};
}

// x: rows of bf16 or fp16, or, with x_scale, of 8-bit integers that quantize_rows made; out_type: of the result in that case
Tensor linear_int8(const std::shared_ptr<Library>& lib, const Tensor& x_in, const std::optional<Tensor>& x_scale_in, const Tensor& w_in, const Tensor& w_scale_in,
                   const std::optional<Tensor>& bias_in, int64_t act_in, const std::optional<Tensor>& gate_in, const std::optional<Tensor>& residual_in, at::ScalarType out_type) {
    const char* const what = "linear_int8";
    const Tensor *xs = address(x_scale_in), *bias = address(bias_in), *gate_p = address(gate_in), *residual_p = address(residual_in);
    begin(*lib, what, x_in, {&x_in, xs, &w_in, &w_scale_in, bias, gate_p, residual_p});
    const int act = activation(what, act_in);
    const int64_t K = row_length(what, x_in);
    auto integers_of = [&](const char* name, const Tensor& t) {
        if (t.scalar_type() != at::kChar) fail(Failure::kValue, std::string(what) + ": " + name + " must be torch.int8 (got " + name_of(t.scalar_type()) + ")");
    };
    auto scales_of = [&](const char* name, const Tensor& t, at::IntArrayRef sizes) {
        if (t.scalar_type() != at::kFloat) fail(Failure::kValue, std::string(what) + ": " + name + " must be torch.float32 (got " + name_of(t.scalar_type()) + ")");
        check_vector(what, name, &t, sizes);
    };
    if (xs != nullptr) {
        integers_of("x", x_in);
        scales_of("the scales of x", *xs, without_last(x_in));
    } else {
        dtype_of(x_in, false, what);
        out_type = x_in.scalar_type();
    }
    integers_of("weight", w_in);
    check_weight(what, "weight", w_in, K, x_in);
    const int64_t N = w_in.size(0);
    scales_of("scale", w_scale_in, {N});
    if (K > LLSA_INT8_MAX_K) fail(Failure::kNotImplemented, "linear_int8 takes at most " + std::to_string(LLSA_INT8_MAX_K) + " channels in (sums of 32 bits; got " + std::to_string(K) + ")");
    for (const Tensor* t : {bias, gate_p, residual_p})
        if (t != nullptr && t->scalar_type() != out_type)
            fail(Failure::kValue, "linear_int8: bias, gate and residual must have the result's dtype, " + name_of(out_type) + " (got " + name_of(t->scalar_type()) + ")");
    check_vector(what, "bias", bias, {N});
    const LayerInputs in = layer_inputs(what, x_in, gate_p, residual_p, N);
    refuse_gradients(what, {&x_in, xs, &w_scale_in, bias, gate_p, residual_p});

    at::AutoDispatchBelowADInplaceOrView below;
    c10::OptionalDeviceGuard guard(lib->device ? std::optional<at::Device>(x_in.device()) : std::nullopt);
    std::vector<int64_t> out_sizes = x_in.sizes().vec();
    out_sizes.back() = N;
    const Tensor out = at::empty(out_sizes, x_in.options().dtype(out_type));
    if (in.rows == 0) return out;
    Call call(*lib, x_in);
    llsa_quantize_args q{};
    q.K = static_cast<int32_t>(K);
    std::vector<Tensor> copied;
    const Rows w = integers(w_in, q, copied);
    Rows x, from;
    Tensor scale;
    bool direct = false;
    if (xs != nullptr) {
        x = integers(x_in, q, copied);
        scale = in_memory(*xs).contiguous();
    } else {
        from = rows_of(x_in);
        // few rows: in one launch with the product, where nothing has to be copied
        direct = q.pads == 0 && from.count <= LLSA_INT8_DIRECT_ROWS && K % 16 == 0 && aligned(from.t) && from.ld % 8 == 0 && from.ld <= (int64_t(1) << 23);
    }
    if (xs == nullptr && !direct) {
        x.t = at::empty({from.count, pad16(K)}, x_in.options().dtype(at::kChar));
        x.ld = pad16(K); x.count = from.count; x.cols = K;
        scale = at::empty({from.count}, x_in.options().dtype(at::kFloat));
        quantize_job(q, from, x.t, scale, dtype_of(x_in, false, what), true);
    }
    if (q.rows > 0 || q.pads > 0) lib->check(lib->quantize_rows(&q, call.stream()), what);
    const Tensor w_scale = in_memory(w_scale_in).contiguous(), b = dense_vector(bias), gate = dense_vector(gate_p);
    const Rows residual = call.addend(residual_p);
    llsa_int8_args a{};
    if (direct) { a.x = from.p(); a.ldx = from.ld; }
    else { a.q = x.p(); a.ldq = x.ld; a.q_scale = scale.data_ptr<float>(); }
    a.w = w.p(); a.ldw = w.ld; a.w_scale = w_scale.data_ptr<float>();
    if (b.defined()) a.bias = b.data_ptr();
    if (gate.defined()) { a.gate = gate.data_ptr(); a.s_gate = gate.size(0) > 1 ? gate.stride(0) : 0; }
    a.residual = residual.p(); a.ldr = residual.ld;
    a.out = out.data_ptr(); a.ldo = N;
    a.M = in.rows; a.per_sample = in.per_sample(); a.N = static_cast<int32_t>(N); a.K = static_cast<int32_t>(K); a.act = act; a.dtype = dtype_of(out, false, what);
    lib->check(lib->linear_int8(&a, call.stream()), what);
    return out;
}

}  // namespace

void bind_int8(py::module_& m) {
    typedef std::shared_ptr<Library> Lib;
    typedef std::optional<Tensor> Optional;
    m.def("quantize_rows", torch::wrap_pybind_function([](const Lib& lib, const Tensor& x) { return without_interpreter([&] { return quantize_rows(lib, x); }); }));
    m.def("linear_int8", torch::wrap_pybind_function([](const Lib& lib, const Tensor& x, const Optional& x_scale, const Tensor& w, const Tensor& w_scale, const Optional& bias, int64_t act,
                                                        const Optional& gate, const Optional& residual, at::ScalarType out_type) {
        return without_interpreter([&] { return linear_int8(lib, x, x_scale, w, w_scale, bias, act, gate, residual, out_type); });
    }));
}
