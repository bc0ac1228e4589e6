// The host side of the operators around the attention (layer_norm, linear, feed_forward): argument checks, the calls of the C ABI, and
// the autograd nodes.  Native for the reason operators.cpp is: a layer norm of 1024 tokens runs for a few microseconds.
#include "block_common.h"

namespace {

using namespace llsa_host;

// ---------------------------------------------------------------------------------------
// layer norm
// ---------------------------------------------------------------------------------------
struct NormInputs {
    Tensor weight, bias, scale, shift;    // as the kernels read them; undefined: none
    int vtype;
};
void norm_inputs(llsa_layer_norm_args& a, const NormInputs& v) {
    a.weight = v.weight.defined() ? v.weight.data_ptr() : nullptr;
    a.bias = v.bias.defined() ? v.bias.data_ptr() : nullptr;
    a.scale = v.scale.defined() ? v.scale.data_ptr() : nullptr;
    a.shift = v.shift.defined() ? v.shift.data_ptr() : nullptr;
    a.s_scale = v.scale.defined() && v.scale.size(0) > 1 ? v.scale.stride(0) : 0;
    a.s_shift = v.shift.defined() && v.shift.size(0) > 1 ? v.shift.stride(0) : 0;
    a.vtype = v.vtype;
}
// elements next to each other, of type `type`; rows of samples may be any step apart
Tensor small_vector(const Tensor* t, at::ScalarType type) {
    if (t == nullptr) return Tensor();
    const Tensor v = in_memory(t->scalar_type() == type ? *t : t->to(type));
    return v.size(-1) <= 1 || v.stride(-1) == 1 ? v : v.contiguous();
}

struct LayerNormBackward : public BlockNode {
    std::vector<int64_t> sizes;
    int64_t rows, per_sample, samples, C;
    bool has[4];                          // weight, bias, scale, shift
    at::ScalarType types[4], vector_type;
    float eps;
    std::string name() const override { return "LayerNormBackward"; }
    variable_list run(const Tensor& grad, const std::vector<Tensor>& saved) override {
        Call call(*lib, grad);
        const Tensor stats = as_kept(saved[1]);
        const Rows x = rows_of(saved[0]), dy = rows_of(grad);
        NormInputs v;
        v.vtype = vector_type == at::kFloat ? LLSA_DTYPE_F32 : dtype_of(saved[0], true, "layer_norm");
        auto again = [&](int i) { return saved[i].defined() ? small_vector(&saved[i], vector_type) : Tensor(); };
        v.weight = again(2); v.bias = again(3); v.scale = again(4);
        llsa_layer_norm_args a{};
        norm_inputs(a, v);
        a.x = x.p(); a.ldx = x.ld; a.dy = dy.p(); a.lddy = dy.ld; a.stats = stats.data_ptr<float>();
        a.rows = rows; a.per_sample = per_sample; a.C = static_cast<int32_t>(C); a.dtype = dtype_of(grad, true, "layer_norm"); a.eps = eps;
        Tensor dx, d[4];
        if (task_should_compute_output(0)) {
            dx = at::empty(sizes, grad.options());
            a.dx = dx.data_ptr(); a.lddx = C;
        }
        size_t at_ = 1;
        bool any = false;
        const auto options = grad.options().dtype(vector_type);
        for (int i = 0; i < 4; i++)
            if (has[i] && task_should_compute_output(at_++)) {
                d[i] = i < 2 ? at::empty({C}, options) : at::empty({samples, C}, options);
                any = true;
            }
        if (rows > 0 && (dx.defined() || any)) {
            Tensor workspace;
            if (any) {
                workspace = call.bytes(lib->layer_norm_bwd_workspace_bytes(rows, per_sample, static_cast<int>(C)));
                a.workspace = workspace.data_ptr();
            }
            auto at_ptr = [](const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; };
            a.dweight = at_ptr(d[0]); a.dbias = at_ptr(d[1]); a.dscale = at_ptr(d[2]); a.dshift = at_ptr(d[3]);
            lib->check(lib->layer_norm_bwd(&a, call.stream()), "layer_norm_bwd");
        }
        variable_list r{dx};
        for (int i = 0; i < 4; i++)
            if (has[i]) {
                if (d[i].defined() && rows == 0) d[i].zero_();
                r.push_back(d[i].defined() && d[i].scalar_type() != types[i] ? d[i].to(types[i]) : d[i]);
            }
        return r;
    }
};

Tensor layer_norm(const std::shared_ptr<Library>& lib, const Tensor& x_in, const std::optional<Tensor>& weight_in, const std::optional<Tensor>& bias_in,
                  const std::optional<Tensor>& scale_in, const std::optional<Tensor>& shift_in, double eps) {
    const Tensor* in[4] = {address(weight_in), address(bias_in), address(scale_in), address(shift_in)};
    begin(*lib, "layer_norm", x_in, {&x_in, in[0], in[1], in[2], in[3]});
    const int dtype = dtype_of(x_in, true, "layer_norm");
    if (x_in.dim() < 1 || x_in.size(-1) < 1 || x_in.size(-1) > LLSA_NORM_MAX_CHANNELS)
        fail(Failure::kNotImplemented, "layer_norm takes rows of 1 to " + std::to_string(LLSA_NORM_MAX_CHANNELS) + " channels (got " + text_of(x_in.sizes()) + ")");
    const int64_t C = x_in.size(-1);
    check_vector("layer_norm", "weight", in[0], {C});
    check_vector("layer_norm", "bias", in[1], {C});
    const bool samples = in[2] != nullptr || in[3] != nullptr;
    const int64_t B = samples ? samples_of("layer_norm", "scale and shift", x_in) : 1;
    check_vector("layer_norm", "scale", in[2], {B, C});
    check_vector("layer_norm", "shift", in[3], {B, C});
    // the small vectors: of the rows' type if they all are, else in fp32
    at::ScalarType vector_type = x_in.scalar_type();
    for (const Tensor* t : in)
        if (t != nullptr && t->scalar_type() != x_in.scalar_type()) {
            if (t->scalar_type() != at::kFloat)
                fail(Failure::kValue, "layer_norm: weight, bias, scale and shift have the rows' dtype or torch.float32 (got " + name_of(t->scalar_type()) + ")");
            vector_type = at::kFloat;
        }
    const bool grad = wants({&x_in, in[0], in[1], in[2], in[3]});
    Tensor y, stats;
    Rows x;
    NormInputs v;
    std::shared_ptr<LayerNormBackward> node;
    {
        at::AutoDispatchBelowADInplaceOrView below;
        c10::OptionalDeviceGuard guard(lib->device ? std::optional<at::Device>(x_in.device()) : std::nullopt);
        x = rows_of(x_in);
        y = at::empty(x_in.sizes(), x_in.options());
        if (grad) stats = at::empty({x.count, 2}, x_in.options().dtype(at::kFloat));
        v.vtype = vector_type == at::kFloat ? LLSA_DTYPE_F32 : dtype;
        v.weight = small_vector(in[0], vector_type); v.bias = small_vector(in[1], vector_type);
        v.scale = small_vector(in[2], vector_type); v.shift = small_vector(in[3], vector_type);
        const int64_t per_sample = std::max<int64_t>(1, samples && B > 0 ? x.count / B : x.count);
        if (x.count > 0) {
            llsa_layer_norm_args a{};
            norm_inputs(a, v);
            a.x = x.p(); a.ldx = x.ld; a.y = y.data_ptr(); a.ldy = C; a.stats = grad ? stats.data_ptr<float>() : nullptr;
            a.rows = x.count; a.per_sample = per_sample; a.C = static_cast<int32_t>(C); a.dtype = dtype; a.eps = static_cast<float>(eps);
            lib->check(lib->layer_norm_fwd(&a, lib->stream(x_in)), "layer_norm_fwd");
        }
        if (grad) {
            node = make_node<LayerNormBackward>(lib);
            node->sizes = x_in.sizes().vec();
            node->rows = x.count; node->per_sample = per_sample; node->samples = B; node->C = C;
            node->vector_type = vector_type;
            node->eps = static_cast<float>(eps);
            for (int i = 0; i < 4; i++) {
                node->has[i] = in[i] != nullptr;
                node->types[i] = in[i] != nullptr ? in[i]->scalar_type() : vector_type;
            }
        }
    }
    if (node) {
        node->set_next_edges(torch::autograd::collect_next_edges(present({&x_in, in[0], in[1], in[2], in[3]})));
        torch::autograd::set_history(y, node);
        node->keep(x.t, x_in);
        node->keep(stats, stats);
        auto keep = [&](const Tensor& t, const Tensor* input) { node->keep(t, input != nullptr ? *input : t); };
        keep(v.weight, in[0]);
        keep(v.bias, in[1]);
        keep(v.scale, in[2]);
    }
    return y;
}

// ---------------------------------------------------------------------------------------
// linear layers
// ---------------------------------------------------------------------------------------
// dz of a layer out of dout: dout itself where there is neither gate nor activation
Rows layer_dz(const Call& call, const Rows& dout_any, const Tensor& dout, const Tensor& gate, const Tensor& z, int64_t per_sample, int act, int dtype, Tensor* dgate) {
    if (act == LLSA_ACT_NONE && !gate.defined()) return call.operand(dout);
    Rows dz;
    dz.t = call.rows(dout_any.count, dout_any.cols);
    dz.ld = dz.t.size(1); dz.count = dout_any.count; dz.cols = dout_any.cols;
    llsa_linear_args a{};
    a.dout = dout_any.p(); a.lddout = dout_any.ld;
    if (gate.defined()) { a.gate = gate.data_ptr(); a.s_gate = gate.size(0) > 1 ? gate.stride(0) : 0; }
    if (z.defined()) { a.z = z.data_ptr(); a.ldz = z.size(1); }
    a.dz_out = dz.p(); a.lddz = dz.ld;
    a.M = dz.count; a.per_sample = per_sample; a.N = static_cast<int32_t>(dz.cols); a.K = 1; a.act = act; a.dtype = dtype;
    Tensor workspace;
    if (dgate != nullptr) {
        *dgate = at::empty({dz.count / per_sample, dz.cols}, dout.options());
        workspace = call.bytes(call.lib().linear_dz_workspace_bytes(dz.count, per_sample, a.N));
        a.dgate = dgate->data_ptr();
        a.workspace = workspace.data_ptr();
    }
    call.lib().check(call.lib().linear_dz(&a, call.stream()), "linear_dz");
    return dz;
}
// Whether the gate of a layer without an activation stays out of the rows in the backward.  It then costs sums and weights of every sample, 12 N K bytes
// each, in place of passes over its rows: dout and the kept x W^T + b in, dz out, that kept in the forward, 10 T N bytes.
bool gate_in_weights(int64_t per_sample, int64_t samples, int64_t K) { return per_sample >= 2 * K && samples <= LLSA_LINEAR_MAX_GATED_SAMPLES; }
// every sample's weights with its gate; behind them, in fp16, a row of scales for each sample
void* scales_of(const Rows& gated, int64_t samples, int dtype) {
    return dtype == LLSA_DTYPE_F16 ? static_cast<char*>(gated.p()) + 2 * samples * gated.count * gated.ld : nullptr;
}
Rows gated_weights(const Call& call, const Rows& w, const Tensor& gate, int64_t samples, int dtype) {
    Rows r;
    r.t = call.rows(samples * (w.count + (dtype == LLSA_DTYPE_F16)), w.cols);
    r.ld = r.t.size(1); r.count = w.count; r.cols = w.cols;
    llsa_linear_args a{};
    a.w = w.p(); a.ldw = w.ld; a.gate = gate.data_ptr(); a.s_gate = gate.size(0) > 1 ? gate.stride(0) : 0;
    a.out = r.p(); a.ldo = r.ld; a.scales = scales_of(r, samples, dtype);
    a.M = samples; a.per_sample = 1; a.N = static_cast<int32_t>(w.count); a.K = static_cast<int32_t>(w.cols); a.dtype = dtype;
    call.lib().check(call.lib().linear_gate_rows(&a, call.stream()), "linear_gate_rows");
    return r;
}
// dx (rows `out`), multiplied by act'(z) if there is a z.  per_sample: of gated weights, else 0
void layer_dx(const Call& call, const Rows& dz, const Rows& w, const Tensor& out, int64_t ldo, const Tensor& z, int act, int dtype, int64_t per_sample = 0) {
    llsa_linear_args a{};
    a.dz = dz.p(); a.lddz = dz.ld; a.w = w.p(); a.ldw = w.ld;
    a.out = out.data_ptr(); a.ldo = ldo;
    if (z.defined()) { a.z = z.data_ptr(); a.ldz = z.size(1); a.act = act; a.padded = 1; }
    if (per_sample > 0) {
        a.s_w = w.count * w.ld;
        a.scales = scales_of(w, dz.count / per_sample, dtype);
    }
    a.M = dz.count; a.per_sample = std::max<int64_t>(1, per_sample); a.N = static_cast<int32_t>(dz.cols); a.K = static_cast<int32_t>(w.cols); a.dtype = dtype;
    call.lib().check(call.lib().linear_dx(&a, call.stream()), "linear_dx");
}
// dw and db; with a gate (that stays out of the rows: dz is dout) also dgate, if `dgate` is defined, for which w and bias are needed
struct Gated {
    Tensor gate, bias, dgate;
    Rows w;
    int64_t per_sample = 1;
};
void layer_dw(const Call& call, const Rows& dz, const Rows& x, const Tensor& dw, const Tensor& db, int dtype, const Gated* gated = nullptr) {
    llsa_linear_args a{};
    a.dz = dz.p(); a.lddz = dz.ld; a.x = x.p(); a.ldx = x.ld;
    a.out = dw.data_ptr(); a.ldo = x.cols;
    if (db.defined()) a.dbias = db.data_ptr();
    a.M = dz.count; a.per_sample = 1; a.N = static_cast<int32_t>(dz.cols); a.K = static_cast<int32_t>(x.cols); a.dtype = dtype;
    if (gated != nullptr) {
        a.gate = gated->gate.data_ptr(); a.s_gate = gated->gate.size(0) > 1 ? gated->gate.stride(0) : 0;
        a.per_sample = gated->per_sample;
        if (gated->dgate.defined()) {
            a.dgate = gated->dgate.data_ptr();
            a.w = gated->w.p(); a.ldw = gated->w.ld;
            if (gated->bias.defined()) a.bias = gated->bias.data_ptr();
        }
    }
    const Tensor workspace = call.bytes(call.lib().linear_dw_workspace_bytes(a.M, gated != nullptr ? a.M / a.per_sample : 1, a.N, a.K));
    a.workspace = workspace.data_ptr();
    call.lib().check(call.lib().linear_dw(&a, call.stream()), "linear_dw");
}
// out (rows of N, contiguous or padded) = residual + gate * act(x W^T + bias); z: where the pre-activation is wanted
void layer_fwd(const Call& call, const Rows& x, const Rows& w, const Tensor& bias, const Tensor& gate, const Rows& residual, const Tensor& z, const Tensor& out, int64_t ldo,
               bool padded, int64_t per_sample, int act, int dtype) {
    llsa_linear_args a{};
    a.x = x.p(); a.ldx = x.ld; a.w = w.p(); a.ldw = w.ld;
    if (bias.defined()) a.bias = bias.data_ptr();
    if (gate.defined()) { a.gate = gate.data_ptr(); a.s_gate = gate.size(0) > 1 ? gate.stride(0) : 0; }
    a.residual = residual.p(); a.ldr = residual.ld;
    a.out = out.data_ptr(); a.ldo = ldo; a.padded = padded;
    if (z.defined()) { a.z = z.data_ptr(); a.ldz = z.size(1); }
    a.M = x.count; a.per_sample = per_sample; a.N = static_cast<int32_t>(w.count); a.K = static_cast<int32_t>(pad8(w.cols)); a.act = act; a.dtype = dtype;
    call.lib().check(call.lib().linear_fwd(&a, call.stream()), "linear_fwd");
}

struct LinearBackward : public BlockNode {
    std::vector<int64_t> sizes;
    int64_t rows, per_sample, samples, K, N;
    bool has_bias, has_gate, has_residual, has_z, gate_out;      // gate_out: the gate stays out of the rows
    int act, dtype;
    std::string name() const override { return "LinearBackward"; }
    variable_list run(const Tensor& grad, const std::vector<Tensor>& saved) override {
        Call call(*lib, grad);
        size_t at_ = 2;
        const bool want_x = task_should_compute_output(0), want_w = task_should_compute_output(1);
        const bool want_b = has_bias && task_should_compute_output(at_++);
        const bool want_g = has_gate && task_should_compute_output(at_++);
        const bool want_r = has_residual && task_should_compute_output(at_);
        Tensor dx, dw, db, dg;
        if (want_x) dx = at::empty(sizes, grad.options());
        if (rows > 0) {
            const Tensor z = has_z ? as_kept(saved[3]) : Tensor();
            const Tensor gate = has_gate ? dense_vector(&saved[2]) : Tensor();
            if (want_x || want_w || want_b || want_g) {
                const Rows dz = gate_out ? call.operand(grad) : layer_dz(call, rows_of(grad), grad, gate, z, per_sample, act, dtype, want_g ? &dg : nullptr);
                const Rows w = want_x || (gate_out && want_g) ? kept_operand(call, saved[1], K) : Rows();
                if (want_x) layer_dx(call, dz, gate_out ? gated_weights(call, w, gate, samples, dtype) : w, dx, K, Tensor(), act, dtype, gate_out ? per_sample : 0);
                if (want_w || want_b || (gate_out && want_g)) {
                    dw = at::empty({N, K}, grad.options());
                    if (want_b) db = at::empty({N}, grad.options());
                    Gated g;
                    if (gate_out) {
                        if (want_g) g.dgate = dg = at::empty({samples, N}, grad.options());
                        g.gate = gate; g.w = w; g.per_sample = per_sample;
                        g.bias = saved[4].defined() ? dense_vector(&saved[4]) : Tensor();
                    }
                    layer_dw(call, dz, kept_operand(call, saved[0], K), dw, db, dtype, gate_out ? &g : nullptr);
                }
            }
        } else {
            if (want_w) dw = zeros_like_weight(N, K, grad);
            if (want_b) db = at::zeros({N}, grad.options());
            if (want_g) dg = at::zeros({samples, N}, grad.options());
        }
        variable_list r{dx, want_w ? dw : Tensor()};
        if (has_bias) r.push_back(db);
        if (has_gate) r.push_back(want_g ? dg : Tensor());
        if (has_residual) r.push_back(want_r ? grad : Tensor());
        return r;
    }
};

Tensor linear(const std::shared_ptr<Library>& lib, const Tensor& x_in, const Tensor& w_in, const std::optional<Tensor>& bias_in, int64_t act_in,
              const std::optional<Tensor>& gate_in, const std::optional<Tensor>& residual_in) {
    const Tensor *bias_p = address(bias_in), *gate_p = address(gate_in), *residual_p = address(residual_in);
    begin(*lib, "linear", x_in, {&x_in, &w_in, bias_p, gate_p, residual_p});
    const int dtype = dtype_of(x_in, false, "linear"), act = activation("linear", act_in);
    if (x_in.dim() < 1) fail(Failure::kValue, "linear: x needs a dimension of channels");
    check_weight("linear", "weight", w_in, x_in.size(-1), x_in);
    const int64_t K = w_in.size(1), N = w_in.size(0);
    same_types("linear", x_in, {&w_in, bias_p, gate_p, residual_p});
    check_vector("linear", "bias", bias_p, {N});
    const LayerInputs in = layer_inputs("linear", x_in, gate_p, residual_p, N);
    const bool grad = wants({&x_in, &w_in, bias_p, gate_p, residual_p});
    const bool inner = grad && wants({&x_in, &w_in, bias_p}), gates = grad && wants({gate_p});
    const bool gate_out = gate_p != nullptr && act == LLSA_ACT_NONE && gate_in_weights(in.per_sample(), in.samples, K);
    std::vector<int64_t> out_sizes = x_in.sizes().vec();
    out_sizes.back() = N;
    Tensor out, z, gate;
    Rows x, w;
    std::shared_ptr<LinearBackward> node;
    {
        at::AutoDispatchBelowADInplaceOrView below;
        c10::OptionalDeviceGuard guard(lib->device ? std::optional<at::Device>(x_in.device()) : std::nullopt);
        Call call(*lib, x_in);
        out = at::empty(out_sizes, x_in.options());
        gate = dense_vector(gate_p);
        if (in.rows > 0) {
            call.operands({{&x_in, &x}, {&w_in, &w}});
            if ((act != LLSA_ACT_NONE && inner) || (gates && !gate_out)) z = call.rows(in.rows, N);
            layer_fwd(call, x, w, dense_vector(bias_p), gate, call.addend(residual_p), z, out, N, false, in.per_sample(), act, dtype);
        } else {
            x.t = x_in;
            w.t = w_in;
        }
        if (grad) {
            node = make_node<LinearBackward>(lib);
            node->sizes = x_in.sizes().vec();
            node->rows = in.rows; node->per_sample = in.per_sample(); node->samples = in.samples; node->K = K; node->N = N;
            node->has_bias = bias_p != nullptr; node->has_gate = gate_p != nullptr; node->has_residual = residual_p != nullptr; node->has_z = z.defined(); node->gate_out = gate_out;
            node->act = act; node->dtype = dtype;
        }
    }
    if (node) {
        node->set_next_edges(torch::autograd::collect_next_edges(present({&x_in, &w_in, bias_p, gate_p, residual_p})));
        torch::autograd::set_history(out, node);
        // (x is needed for the gradient of the weight, the weight for that of x; each as the products read it)
        node->keep(wants({&w_in, bias_p}) || (gates && gate_out) ? x.t : Tensor(), x_in);
        node->keep(x_in.requires_grad() || (gates && gate_out) ? w.t : Tensor(), w_in);
        node->keep(gate, gate_p != nullptr ? *gate_p : gate);
        node->keep(z, z);
        node->keep(gates && gate_out && bias_p != nullptr ? *bias_p : Tensor(), bias_p != nullptr ? *bias_p : Tensor());
    }
    return out;
}

// ---------------------------------------------------------------------------------------
// feed-forward block
// ---------------------------------------------------------------------------------------
struct FeedForwardBackward : public BlockNode {
    std::vector<int64_t> sizes;
    int64_t rows, per_sample, samples, C, F, N;
    bool has_b1, has_b2, has_gate, has_residual, has_y, gate_out;
    int act, dtype;
    std::string name() const override { return "FeedForwardBackward"; }
    variable_list run(const Tensor& grad, const std::vector<Tensor>& saved) override {
        Call call(*lib, grad);
        size_t at_ = 1;
        const bool want_x = task_should_compute_output(0), want_w1 = task_should_compute_output(at_++);
        const bool want_b1 = has_b1 && task_should_compute_output(at_++), want_w2 = task_should_compute_output(at_++);
        const bool want_b2 = has_b2 && task_should_compute_output(at_++), want_g = has_gate && task_should_compute_output(at_++);
        const bool want_r = has_residual && task_should_compute_output(at_);
        const bool inner = want_x || want_w1 || want_b1, outer = want_w2 || want_b2;
        Tensor dx, dw1, db1, dw2, db2, dg;
        if (want_x) dx = at::empty(sizes, grad.options());
        const auto o = grad.options();
        if (rows > 0 && (inner || outer || want_g)) {
            const Tensor gate = has_gate ? dense_vector(&saved[3]) : Tensor();
            const Tensor y = has_y ? as_kept(saved[6]) : Tensor();
            const Rows dz2 = gate_out ? call.operand(grad) : layer_dz(call, rows_of(grad), grad, gate, y, per_sample, LLSA_ACT_NONE, dtype, want_g ? &dg : nullptr);
            const Rows w2 = inner || (gate_out && want_g) ? kept_operand(call, saved[2], F) : Rows();
            if (outer || (gate_out && want_g)) {
                Rows h;
                h.t = as_kept(saved[5]);
                h.ld = h.t.size(1); h.count = rows; h.cols = F;
                dw2 = at::empty({N, F}, o);
                if (want_b2) db2 = at::empty({N}, o);
                Gated g;
                if (gate_out) {
                    if (want_g) g.dgate = dg = at::empty({samples, N}, o);
                    g.gate = gate; g.w = w2; g.per_sample = per_sample;
                    g.bias = saved[7].defined() ? dense_vector(&saved[7]) : Tensor();
                }
                layer_dw(call, dz2, h, dw2, db2, dtype, gate_out ? &g : nullptr);
            }
            if (inner) {
                Rows dz1;
                dz1.t = call.rows(rows, F);
                dz1.ld = dz1.t.size(1); dz1.count = rows; dz1.cols = F;
                layer_dx(call, dz2, gate_out ? gated_weights(call, w2, gate, samples, dtype) : w2, dz1.t, dz1.ld, as_kept(saved[4]), act, dtype,
                         gate_out ? per_sample : 0);
                if (want_x) layer_dx(call, dz1, kept_operand(call, saved[1], C), dx, C, Tensor(), act, dtype);
                if (want_w1 || want_b1) {
                    dw1 = at::empty({F, C}, o);
                    if (want_b1) db1 = at::empty({F}, o);
                    layer_dw(call, dz1, kept_operand(call, saved[0], C), dw1, db1, dtype);
                }
            }
        } else if (rows == 0) {
            if (want_w1) dw1 = zeros_like_weight(F, C, grad);
            if (want_b1) db1 = at::zeros({F}, o);
            if (want_w2) dw2 = zeros_like_weight(N, F, grad);
            if (want_b2) db2 = at::zeros({N}, o);
            if (want_g) dg = at::zeros({samples, N}, o);
        }
        variable_list r{dx, want_w1 ? dw1 : Tensor()};
        if (has_b1) r.push_back(db1);
        r.push_back(want_w2 ? dw2 : Tensor());
        if (has_b2) r.push_back(db2);
        if (has_gate) r.push_back(want_g ? dg : Tensor());
        if (has_residual) r.push_back(want_r ? grad : Tensor());
        return r;
    }
};

Tensor feed_forward(const std::shared_ptr<Library>& lib, const Tensor& x_in, const Tensor& w1_in, const std::optional<Tensor>& b1_in, const Tensor& w2_in,
                    const std::optional<Tensor>& b2_in, int64_t act_in, const std::optional<Tensor>& gate_in, const std::optional<Tensor>& residual_in) {
    const char* const what = "feed_forward";
    const Tensor *b1 = address(b1_in), *b2 = address(b2_in), *gate_p = address(gate_in), *residual_p = address(residual_in);
    begin(*lib, what, x_in, {&x_in, &w1_in, b1, &w2_in, b2, gate_p, residual_p});
    const int dtype = dtype_of(x_in, false, what), act = activation(what, act_in);
    if (act == LLSA_ACT_NONE) fail(Failure::kValue, "feed_forward needs an activation");
    if (x_in.dim() < 1) fail(Failure::kValue, "feed_forward: x needs a dimension of channels");
    check_weight(what, "w_in", w1_in, x_in.size(-1), x_in);
    check_weight(what, "w_out", w2_in, w1_in.size(0), x_in);
    const int64_t C = w1_in.size(1), F = w1_in.size(0), N = w2_in.size(0);
    same_types(what, x_in, {&w1_in, b1, &w2_in, b2, gate_p, residual_p});
    check_vector(what, "b_in", b1, {F});
    check_vector(what, "b_out", b2, {N});
    const LayerInputs in = layer_inputs(what, x_in, gate_p, residual_p, N);
    const bool grad = wants({&x_in, &w1_in, b1, &w2_in, b2, gate_p, residual_p});
    const bool inner = grad && wants({&x_in, &w1_in, b1}), outer = grad && wants({&w2_in, b2}), gates = grad && wants({gate_p});
    const bool gate_out = gate_p != nullptr && gate_in_weights(in.per_sample(), in.samples, F);
    std::vector<int64_t> out_sizes = x_in.sizes().vec();
    out_sizes.back() = N;
    Tensor out, z, h, y, gate;
    Rows x, w1, w2;
    std::shared_ptr<FeedForwardBackward> node;
    {
        at::AutoDispatchBelowADInplaceOrView below;
        c10::OptionalDeviceGuard guard(lib->device ? std::optional<at::Device>(x_in.device()) : std::nullopt);
        Call call(*lib, x_in);
        out = at::empty(out_sizes, x_in.options());
        gate = dense_vector(gate_p);
        if (in.rows > 0) {
            Rows hidden;
            call.operands({{&x_in, &x}, {&w1_in, &w1}, {&w2_in, &w2}});
            h = call.rows(in.rows, F);
            hidden.t = h; hidden.ld = h.size(1); hidden.count = in.rows; hidden.cols = F;
            if (inner) z = call.rows(in.rows, F);
            if (gates && !gate_out) y = call.rows(in.rows, N);
            layer_fwd(call, x, w1, dense_vector(b1), Tensor(), Rows(), z, h, hidden.ld, true, 1, act, dtype);
            layer_fwd(call, hidden, w2, dense_vector(b2), gate, call.addend(residual_p), y, out, N, false, in.per_sample(),
                      LLSA_ACT_NONE, dtype);
        }
        if (grad) {
            node = make_node<FeedForwardBackward>(lib);
            node->sizes = x_in.sizes().vec();
            node->rows = in.rows; node->per_sample = in.per_sample(); node->samples = in.samples; node->C = C; node->F = F; node->N = N;
            node->has_b1 = b1 != nullptr; node->has_b2 = b2 != nullptr; node->has_gate = gate_p != nullptr; node->has_residual = residual_p != nullptr;
            node->has_y = y.defined(); node->gate_out = gate_out;
            node->act = act; node->dtype = dtype;
        }
    }
    if (node) {
        node->set_next_edges(torch::autograd::collect_next_edges(present({&x_in, &w1_in, b1, &w2_in, b2, gate_p, residual_p})));
        torch::autograd::set_history(out, node);
        node->keep(wants({&w1_in, b1}) ? x.t : Tensor(), x_in);
        node->keep(wants({&x_in}) ? w1.t : Tensor(), w1_in);
        node->keep(inner || (gates && gate_out) ? w2.t : Tensor(), w2_in);
        node->keep(gate, gate_p != nullptr ? *gate_p : gate);
        node->keep(z, z);
        node->keep(outer || (gates && gate_out) ? h : Tensor(), h);
        node->keep(y, y);
        node->keep(gates && gate_out && b2 != nullptr ? *b2 : Tensor(), b2 != nullptr ? *b2 : Tensor());
    }
    return out;
}

}  // namespace

void bind_block(py::module_& m) {
    typedef std::shared_ptr<Library> Lib;
    typedef std::optional<Tensor> Optional;
    m.def("layer_norm", torch::wrap_pybind_function([](const Lib& lib, const Tensor& x, const Optional& weight, const Optional& bias, const Optional& scale, const Optional& shift,
                                                       double eps) { return without_interpreter([&] { return layer_norm(lib, x, weight, bias, scale, shift, eps); }); }));
    m.def("linear", torch::wrap_pybind_function([](const Lib& lib, const Tensor& x, const Tensor& w, const Optional& bias, int64_t act, const Optional& gate, const Optional& residual) {
        return without_interpreter([&] { return linear(lib, x, w, bias, act, gate, residual); });
    }));
    m.def("feed_forward", torch::wrap_pybind_function([](const Lib& lib, const Tensor& x, const Tensor& w1, const Optional& b1, const Tensor& w2, const Optional& b2, int64_t act,
                                                         const Optional& gate, const Optional& residual) {
        return without_interpreter([&] { return feed_forward(lib, x, w1, b1, w2, b2, act, gate, residual); });
    }));
}
