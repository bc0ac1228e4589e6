// The host side of rows that choose their weights (route_tokens, grouped_linear, expert_feed_forward): argument checks, the calls of the C ABI, and the
// autograd nodes.
#include "block_common.h"

namespace {

int64_t rows_in(const Tensor& x) {                            // of the last dimension; also where that has none
    int64_t n = 1;
    for (int64_t d = 0; d + 1 < x.dim(); d++) n *= x.size(d);
    return n;
}
std::vector<int64_t> with_last(const Tensor& x, int64_t last) {
    std::vector<int64_t> s = x.sizes().vec();
    s.back() = last;
    return s;
}
Tensor contiguous(const Tensor& t) { return in_memory(t).contiguous(); }

// ---------------------------------------------------------------------------------------
// the router
// ---------------------------------------------------------------------------------------
struct RouteBackward : public BlockNode {
    std::vector<int64_t> sizes;
    int64_t rows, E, k;
    bool normalize;
    int dtype;
    at::ScalarType type;
    std::string name() const override { return "RouteTokensBackward"; }
    variable_list run(const Tensor& grad, const std::vector<Tensor>& saved) override {
        if (!task_should_compute_output(0)) return {Tensor()};
        const Tensor dlogits = at::empty(sizes, grad.options().dtype(type)), dweights = contiguous(grad), experts = contiguous(saved[1]);
        const Rows logits = rows_of(saved[0]);
        llsa_route_args a{};
        a.logits = logits.p(); a.ld = logits.ld; a.experts = experts.data_ptr<int32_t>(); a.dweights = dweights.data_ptr<float>(); a.dlogits = dlogits.data_ptr();
        a.M = rows; a.E = static_cast<int32_t>(E); a.k = static_cast<int32_t>(k); a.normalize = normalize; a.dtype = dtype;
        lib->check(lib->route_tokens_bwd(&a, lib->stream(grad)), "route_tokens_bwd");
        return {dlogits};
    }
};

std::tuple<Tensor, Tensor, Tensor, Tensor, Tensor> route_tokens(const std::shared_ptr<Library>& lib, const Tensor& logits_in, int64_t k, bool normalize) {
    const char* const what = "route_tokens";
    begin(*lib, what, logits_in, {&logits_in});
    const int dtype = dtype_of(logits_in, true, what);
    if (logits_in.dim() < 1 || logits_in.size(-1) < 1 || logits_in.size(-1) > LLSA_MAX_EXPERTS)
        fail(Failure::kNotImplemented, "route_tokens takes logits of 1 to " + std::to_string(LLSA_MAX_EXPERTS) + " experts (got " + text_of(logits_in.sizes()) + ")");
    const int64_t E = logits_in.size(-1), M = rows_in(logits_in);
    if (k < 1 || k > std::min<int64_t>(E, LLSA_MAX_CHOICES))
        fail(Failure::kValue, "route_tokens: experts_per_token must be 1 to " + std::to_string(std::min<int64_t>(E, LLSA_MAX_CHOICES)) + " (got " + std::to_string(k) + ")");
    if (M > LLSA_MAX_SLOTS / k) fail(Failure::kValue, "route_tokens: too many tokens (" + std::to_string(M) + ")");
    const bool grad = wants({&logits_in});
    Tensor weights, experts, order, offsets, places;
    Rows logits;
    std::shared_ptr<RouteBackward> node;
    {
        at::AutoDispatchBelowADInplaceOrView below;
        c10::OptionalDeviceGuard guard(lib->device ? std::optional<at::Device>(logits_in.device()) : std::nullopt);
        Call call(*lib, logits_in);
        const auto ints = logits_in.options().dtype(at::kInt);
        const std::vector<int64_t> chosen = with_last(logits_in, k);
        weights = at::empty(chosen, logits_in.options().dtype(at::kFloat));
        experts = at::empty(chosen, ints);
        order = at::empty({M * k}, ints);
        offsets = M > 0 ? at::empty({E + 1}, ints) : at::zeros({E + 1}, ints);
        places = at::empty(chosen, ints);
        logits = rows_of(logits_in);
        if (M > 0) {
            const Tensor workspace = call.bytes(lib->route_workspace_bytes(M, static_cast<int>(E), static_cast<int>(k)));
            llsa_route_args a{};
            a.logits = logits.p(); a.ld = logits.ld; a.weights = weights.data_ptr<float>(); a.experts = experts.data_ptr<int32_t>(); a.order = order.data_ptr<int32_t>();
            a.offsets = offsets.data_ptr<int32_t>(); a.places = places.data_ptr<int32_t>(); a.workspace = workspace.defined() ? workspace.data_ptr() : nullptr;
            a.M = M; a.E = static_cast<int32_t>(E); a.k = static_cast<int32_t>(k); a.normalize = normalize; a.dtype = dtype;
            lib->check(lib->route_tokens(&a, call.stream()), what);
        }
        if (grad) {
            node = make_node<RouteBackward>(lib);
            node->sizes = logits_in.sizes().vec();
            node->rows = M; node->E = E; node->k = k; node->normalize = normalize; node->dtype = dtype; node->type = logits_in.scalar_type();
        }
    }
    if (node) {
        node->set_next_edges(torch::autograd::collect_next_edges(present({&logits_in})));
        torch::autograd::set_history(weights, node);
        node->keep(logits.t, logits_in);
        node->keep(experts, experts);
    }
    return {weights, experts, order, offsets, places};
}

// ---------------------------------------------------------------------------------------
// products by expert
// ---------------------------------------------------------------------------------------
void check_expert_weight(const char* what, const char* name, const Tensor& w, int64_t experts, int64_t in) {
    if (w.dim() != 3 || w.size(0) < 1 || w.size(1) < 1 || w.size(2) < 1 || (in >= 0 && w.size(2) != in) || (experts >= 0 && w.size(0) != experts))
        fail(Failure::kValue, std::string(what) + ": " + name + " must be (" + (experts >= 0 ? std::to_string(experts) : std::string("experts")) + ", channels out, " +
                                  (in >= 0 ? std::to_string(in) : std::string("channels in")) + ") (got " + text_of(w.sizes()) + ")");
    if (w.size(0) > LLSA_MAX_EXPERTS) fail(Failure::kNotImplemented, std::string(what) + " takes at most " + std::to_string(LLSA_MAX_EXPERTS) + " experts (got " + std::to_string(w.size(0)) + ")");
    if (w.size(1) >= (1 << 23) || w.size(2) >= (1 << 23)) fail(Failure::kValue, std::string(what) + ": too many channels");
    if (w.size(1) * pad8(w.size(2)) >= (int64_t(1) << 31)) fail(Failure::kValue, std::string(what) + ": too many weights of an expert");
    if (w.size(0) * w.size(1) >= (int64_t(1) << 31)) fail(Failure::kValue, std::string(what) + ": too many channels of all experts");
}
void check_ints(const char* what, const char* name, const Tensor& t, at::IntArrayRef sizes) {
    if (t.scalar_type() != at::kInt) fail(Failure::kValue, std::string(what) + ": " + name + " must be torch.int32 (got " + name_of(t.scalar_type()) + ")");
    check_vector(what, name, &t, sizes);
}
void check_rows(const char* what, int64_t rows) {
    if (rows > LLSA_MAX_SLOTS) fail(Failure::kValue, std::string(what) + ": too many rows (" + std::to_string(rows) + ")");
}
// (E, N, K) as rows of the products, which may be copies
struct Weights {
    Rows rows;
    int64_t E, N, K;
    const void* p() const { return rows.p(); }
};
Weights weights_of(const Call& call, const Tensor& w, int64_t E, int64_t N, int64_t K) { return {call.operand(w), E, N, K}; }
void set_weights(llsa_experts_args& a, const Weights& w) {
    a.w = w.p(); a.ldw = w.rows.ld; a.E = static_cast<int32_t>(w.E); a.N = static_cast<int32_t>(w.N); a.K = static_cast<int32_t>(w.K);
}
const int32_t* ints(const Tensor& t) { return t.data_ptr<int32_t>(); }
// act'(z) as a forward keeps it
Tensor slopes_of(const Call& call, int64_t rows, int64_t cols) {
    const Tensor like = call.rows(0, 8);
    return at::empty({rows, pad8(cols)}, like.options().dtype(at::kShort));
}
// rows of fp32 that are added up
Tensor wide_rows(const Call& call, int64_t rows, int64_t cols) {
    const Tensor like = call.rows(0, 8);
    return at::empty({rows, pad8(cols)}, like.options().dtype(at::kFloat));
}
Tensor dense_bias(const Tensor* t) { return t != nullptr ? contiguous(*t) : Tensor(); }

struct GroupedLinearBackward : public BlockNode {
    std::vector<int64_t> sizes;
    int64_t rows, E, N, K;
    bool has_bias;
    int act, dtype;
    std::string name() const override { return "GroupedLinearBackward"; }
    variable_list run(const Tensor& grad, const std::vector<Tensor>& saved) override {
        Call call(*lib, grad);
        const bool want_x = task_should_compute_output(0), want_w = task_should_compute_output(1), want_b = has_bias && task_should_compute_output(2);
        const auto o = grad.options();
        Tensor dx, dw, db;
        if (want_x) dx = at::empty(sizes, o);
        if (rows > 0 && (want_x || want_w || want_b)) {
            const Tensor offsets = contiguous(saved[2]);
            Rows dz;
            if (act == LLSA_ACT_NONE) {
                dz = call.operand(grad);
            } else {
                const Rows dout = rows_of(grad);
                const Tensor slopes = as_kept(saved[3]);
                dz.t = call.rows(rows, N); dz.ld = dz.t.size(1); dz.count = rows; dz.cols = N;
                llsa_experts_args a{};
                a.dz = dout.p(); a.lddz = dout.ld; a.slopes = slopes.data_ptr(); a.ldz = slopes.size(1); a.out = dz.p(); a.ldo = dz.ld; a.offsets = ints(offsets);
                a.rows = rows; a.tokens = rows; a.k = 1; a.E = static_cast<int32_t>(E); a.N = static_cast<int32_t>(N); a.K = 8; a.dtype = dtype;
                lib->check(lib->experts_dz(&a, call.stream()), "experts_dz");
            }
            llsa_experts_args a{};
            a.offsets = ints(offsets); a.rows = rows; a.tokens = rows; a.k = 1; a.dtype = dtype; a.act = LLSA_ACT_NONE;
            a.dz = dz.p(); a.lddz = dz.ld;
            if (want_x) {
                const Weights w = weights_of(call, saved[1], E, N, K);
                llsa_experts_args d = a;
                set_weights(d, w);
                d.out = dx.data_ptr(); d.ldo = K; d.gaps = 1;
                lib->check(lib->experts_dx(&d, call.stream()), "experts_dx");
            }
            if (want_w || want_b) {
                const Rows x = kept_operand(call, saved[0], K);
                dw = at::empty({E, N, K}, o);
                if (want_b) db = at::empty({E, N}, o);
                llsa_experts_args d = a;
                d.E = static_cast<int32_t>(E); d.N = static_cast<int32_t>(N); d.K = static_cast<int32_t>(K);
                d.x = x.p(); d.ldx = x.ld; d.out = dw.data_ptr();
                if (want_b) d.dbias = db.data_ptr();
                const Tensor workspace = call.bytes(lib->experts_dw_workspace_bytes(rows, d.E, d.N, d.K));
                d.workspace = workspace.data_ptr();
                lib->check(lib->experts_dw(&d, call.stream()), "experts_dw");
            }
        } else if (rows == 0) {
            if (want_w) dw = at::zeros({E, N, K}, o);
            if (want_b) db = at::zeros({E, N}, o);
        }
        variable_list r{dx, want_w ? dw : Tensor()};
        if (has_bias) r.push_back(db);
        return r;
    }
};

Tensor grouped_linear(const std::shared_ptr<Library>& lib, const Tensor& x_in, const Tensor& w_in, const Tensor& offsets_in, const std::optional<Tensor>& bias_in, int64_t act_in) {
    const char* const what = "grouped_linear";
    const Tensor* bias_p = address(bias_in);
    begin(*lib, what, x_in, {&x_in, &w_in, &offsets_in, bias_p});
    const int dtype = dtype_of(x_in, false, what), act = activation(what, act_in);
    if (x_in.dim() != 2 || x_in.size(1) < 1) fail(Failure::kValue, "grouped_linear: x must be (rows, channels in) (got " + text_of(x_in.sizes()) + ")");
    check_expert_weight(what, "weight", w_in, -1, x_in.size(1));
    const int64_t rows = x_in.size(0), E = w_in.size(0), N = w_in.size(1), K = w_in.size(2);
    check_ints(what, "offsets", offsets_in, {E + 1});
    same_types(what, x_in, {&w_in, bias_p});
    check_vector(what, "bias", bias_p, {E, N});
    check_rows(what, rows);
    const bool grad = wants({&x_in, &w_in, bias_p});
    Tensor out, slopes, offsets;
    Rows x;
    Weights w;
    std::shared_ptr<GroupedLinearBackward> node;
    {
        at::AutoDispatchBelowADInplaceOrView below;
        c10::OptionalDeviceGuard guard(lib->device ? std::optional<at::Device>(x_in.device()) : std::nullopt);
        Call call(*lib, x_in);
        out = at::empty({rows, N}, x_in.options());
        offsets = contiguous(offsets_in);
        w.rows.t = w_in;
        x.t = x_in;
        if (rows > 0) {
            call.operands({{&x_in, &x}, {&w_in, &w.rows}});
            w.E = E; w.N = N; w.K = pad8(K);
            if (act != LLSA_ACT_NONE && grad) slopes = slopes_of(call, rows, N);
            const Tensor bias = dense_bias(bias_p);
            llsa_experts_args a{};
            set_weights(a, w);
            a.x = x.p(); a.ldx = x.ld; a.offsets = ints(offsets); a.bias = bias.defined() ? bias.data_ptr() : nullptr;
            a.out = out.data_ptr(); a.ldo = N; a.gaps = 1;
            if (slopes.defined()) { a.slopes = slopes.data_ptr(); a.ldz = slopes.size(1); }
            a.rows = rows; a.tokens = rows; a.k = 1; a.act = act; a.dtype = dtype;
            lib->check(lib->experts_fwd(&a, call.stream()), what);
        }
        if (grad) {
            node = make_node<GroupedLinearBackward>(lib);
            node->sizes = x_in.sizes().vec();
            node->rows = rows; node->E = E; node->N = N; node->K = K; node->has_bias = bias_p != nullptr; node->act = act; node->dtype = dtype;
        }
    }
    if (node) {
        node->set_next_edges(torch::autograd::collect_next_edges(present({&x_in, &w_in, bias_p})));
        torch::autograd::set_history(out, node);
        node->keep(wants({&w_in, bias_p}) ? x.t : Tensor(), x_in);
        node->keep(x_in.requires_grad() ? w.rows.t : Tensor(), w_in);
        node->keep(offsets, offsets_in);
        node->keep(slopes, slopes);
    }
    return out;
}

// ---------------------------------------------------------------------------------------
// the routed feed-forward block
// ---------------------------------------------------------------------------------------
// Rows of tokens in the order of the places, multiplied by the router's weights and the gate unless they are NULL
Rows gathered(const Call& call, const Rows& x, const llsa_experts_args& base, const float* weights, const Tensor& gate, int64_t per_sample) {
    Rows r;
    r.t = call.rows(base.rows, x.cols); r.ld = r.t.size(1); r.count = base.rows; r.cols = x.cols;
    llsa_experts_args a = base;
    a.act = LLSA_ACT_NONE;
    a.x = x.p(); a.ldx = x.ld; a.out = r.p(); a.ldo = r.ld; a.weights = weights; a.N = static_cast<int32_t>(x.cols); a.K = 8;
    if (gate.defined()) { a.gate = gate.data_ptr(); a.s_gate = gate.size(0) > 1 ? gate.stride(0) : 0; a.per_sample = per_sample; }
    call.lib().check(call.lib().experts_gather(&a, call.stream()), "experts_gather");
    return r;
}
struct ExpertFeedForwardBackward : public BlockNode {
    std::vector<int64_t> sizes, chosen;   // of x, of the router's weights
    int64_t tokens, k, per_sample, samples, E, C, F, N;
    bool has_b1, has_b2, has_gate, has_residual;
    int dtype;
    enum { kX, kW1, kW2, kGate, kOffsets, kOrder, kPlaces, kWeights, kSlopes, kH, kY };
    std::string name() const override { return "ExpertFeedForwardBackward"; }
    variable_list run(const Tensor& grad, const std::vector<Tensor>& saved) override {
        Call call(*lib, grad);
        size_t at_ = 2;
        const bool want_x = task_should_compute_output(0), want_p = task_should_compute_output(1), want_w1 = task_should_compute_output(at_++);
        const bool want_b1 = has_b1 && task_should_compute_output(at_++), want_w2 = task_should_compute_output(at_++);
        const bool want_b2 = has_b2 && task_should_compute_output(at_++), want_g = has_gate && task_should_compute_output(at_++);
        const bool want_r = has_residual && task_should_compute_output(at_);
        const bool inner = want_x || want_w1 || want_b1, outer = want_w2 || want_b2;
        const auto o = grad.options();
        const int64_t rows = tokens * k;
        Tensor dx, dp, dw1, db1, dw2, db2, dg;
        if (want_x) dx = at::empty(sizes, o);
        if (want_p) dp = at::empty(chosen, o.dtype(at::kFloat));
        if (rows > 0 && (inner || outer || want_p || want_g)) {
            const Rows dout = rows_of(grad);
            const Tensor gate = has_gate ? dense_vector(&saved[kGate]) : Tensor();
            const Tensor places = contiguous(saved[kPlaces]), weights = contiguous(saved[kWeights]);
            llsa_experts_args base{};
            base.places = ints(places); base.rows = rows; base.tokens = tokens; base.k = static_cast<int32_t>(k); base.E = static_cast<int32_t>(E); base.dtype = dtype;
            const Tensor offsets = contiguous(saved[kOffsets]), order = contiguous(saved[kOrder]);
            base.offsets = ints(offsets); base.order = ints(order);
            if (want_p || want_g) {
                const Tensor y = as_kept(saved[kY]);
                Tensor workspace;
                llsa_experts_args a = base;
                a.dz = dout.p(); a.lddz = dout.ld; a.x = y.data_ptr(); a.ldx = y.size(1); a.weights = weights.data_ptr<float>(); a.N = static_cast<int32_t>(N); a.K = 8;
                if (want_p) a.dweights = dp.data_ptr<float>();
                if (has_gate) { a.gate = gate.data_ptr(); a.s_gate = gate.size(0) > 1 ? gate.stride(0) : 0; a.per_sample = per_sample; }
                if (want_g) {
                    dg = at::empty({samples, N}, o);
                    workspace = call.bytes(lib->experts_dweights_workspace_bytes(tokens, per_sample, a.N));
                    a.dgate = dg.data_ptr(); a.workspace = workspace.data_ptr();
                }
                lib->check(lib->experts_dweights(&a, call.stream()), "experts_dweights");
            }
            if (!inner && !outer) return results(dx, dp, dw1, db1, dw2, db2, dg, grad, want_w1, want_w2, want_r);
            const Rows g = gathered(call, dout, base, weights.data_ptr<float>(), gate, per_sample);      // w gate dout
            Rows dz;
            if (inner) {                                      // dz = act'(z) (g W_out)
                const Weights w2 = weights_of(call, saved[kW2], E, N, F);
                const Tensor slopes = as_kept(saved[kSlopes]);
                dz.t = call.rows(rows, F); dz.ld = dz.t.size(1); dz.count = rows; dz.cols = F;
                llsa_experts_args a = base;
                set_weights(a, w2);
                a.dz = g.p(); a.lddz = g.ld;
                a.out = dz.p(); a.ldo = dz.ld; a.padded = 1; a.slopes = slopes.data_ptr(); a.ldz = slopes.size(1);
                lib->check(lib->experts_dx(&a, call.stream()), "experts_dx");
            }
            auto weights_back = [&](const Rows& dz_rows, const Tensor& x, int64_t n, int64_t kk, Tensor& dw, Tensor& db, bool want_bias) {
                dw = at::empty({E, n, kk}, o);
                if (want_bias) db = at::empty({E, n}, o);
                llsa_experts_args a = base;
                a.dz = dz_rows.p(); a.lddz = dz_rows.ld; a.x = x.data_ptr(); a.ldx = x.size(1);
                a.N = static_cast<int32_t>(n); a.K = static_cast<int32_t>(kk); a.out = dw.data_ptr();
                if (want_bias) a.dbias = db.data_ptr();
                const Tensor workspace = call.bytes(lib->experts_dw_workspace_bytes(rows, a.E, a.N, a.K));
                a.workspace = workspace.data_ptr();
                lib->check(lib->experts_dw(&a, call.stream()), "experts_dw");
            };
            if (outer) {
                weights_back(g, as_kept(saved[kH]), N, F, dw2, db2, want_b2);
            }
            if (want_w1 || want_b1) {
                weights_back(dz, as_kept(saved[kX]), F, C, dw1, db1, want_b1);
            }
            if (want_x) {
                const Weights w1 = weights_of(call, saved[kW1], E, F, C);
                const Tensor each = wide_rows(call, rows, C);
                llsa_experts_args a = base;
                set_weights(a, w1);
                a.dz = dz.p(); a.lddz = dz.ld; a.out = each.data_ptr(); a.ldo = each.size(1); a.padded = 1; a.wide = 1; a.gaps = 1;
                lib->check(lib->experts_dx(&a, call.stream()), "experts_dx");
                llsa_experts_args s = base;
                s.x = each.data_ptr(); s.ldx = each.size(1); s.out = dx.data_ptr(); s.ldo = C; s.N = static_cast<int32_t>(C); s.K = 8;
                lib->check(lib->experts_combine(&s, call.stream()), "experts_combine");
            }
        } else if (rows == 0) {
            if (want_w1) dw1 = at::zeros({E, F, C}, o);
            if (want_b1) db1 = at::zeros({E, F}, o);
            if (want_w2) dw2 = at::zeros({E, N, F}, o);
            if (want_b2) db2 = at::zeros({E, N}, o);
            if (want_g) dg = at::zeros({samples, N}, o);
        }
        return results(dx, dp, dw1, db1, dw2, db2, dg, grad, want_w1, want_w2, want_r);
    }
    variable_list results(const Tensor& dx, const Tensor& dp, const Tensor& dw1, const Tensor& db1, const Tensor& dw2, const Tensor& db2, const Tensor& dg, const Tensor& grad, bool want_w1,
                          bool want_w2, bool want_r) const {
        variable_list r{dx, dp, want_w1 ? dw1 : Tensor()};
        if (has_b1) r.push_back(db1);
        r.push_back(want_w2 ? dw2 : Tensor());
        if (has_b2) r.push_back(db2);
        if (has_gate) r.push_back(dg);
        if (has_residual) r.push_back(want_r ? grad : Tensor());
        return r;
    }
};

Tensor expert_feed_forward(const std::shared_ptr<Library>& lib, const Tensor& x_in, const Tensor& weights_in, const Tensor& experts_in, const Tensor& order_in, const Tensor& offsets_in,
                           const Tensor& places_in, const Tensor& w1_in, const std::optional<Tensor>& b1_in, const Tensor& w2_in, const std::optional<Tensor>& b2_in, int64_t act_in,
                           const std::optional<Tensor>& gate_in, const std::optional<Tensor>& residual_in) {
    const char* const what = "expert_feed_forward";
    const Tensor *b1 = address(b1_in), *b2 = address(b2_in), *gate_p = address(gate_in), *residual_p = address(residual_in);
    begin(*lib, what, x_in, {&x_in, &weights_in, &experts_in, &order_in, &offsets_in, &places_in, &w1_in, b1, &w2_in, b2, gate_p, residual_p});
    const int dtype = dtype_of(x_in, false, what), act = activation(what, act_in);
    if (act == LLSA_ACT_NONE) fail(Failure::kValue, "expert_feed_forward needs an activation");
    if (x_in.dim() < 1 || x_in.size(-1) < 1) fail(Failure::kValue, "expert_feed_forward: x needs a dimension of channels");
    check_expert_weight(what, "w_in", w1_in, -1, x_in.size(-1));
    const int64_t E = w1_in.size(0), F = w1_in.size(1), C = w1_in.size(2);
    check_expert_weight(what, "w_out", w2_in, E, F);
    const int64_t N = w2_in.size(1);
    same_types(what, x_in, {&w1_in, b1, &w2_in, b2, gate_p, residual_p});
    check_vector(what, "b_in", b1, {E, F});
    check_vector(what, "b_out", b2, {E, N});
    const LayerInputs in = layer_inputs(what, x_in, gate_p, residual_p, N);
    // the router's results
    if (weights_in.dim() != x_in.dim() || weights_in.size(-1) < 1 || weights_in.size(-1) > LLSA_MAX_CHOICES)
        fail(Failure::kValue, "expert_feed_forward: the routing must be of x's tokens, 1 to " + std::to_string(LLSA_MAX_CHOICES) + " experts each (got weights " + text_of(weights_in.sizes()) + " for x " + text_of(x_in.sizes()) + ")");
    const int64_t k = weights_in.size(-1), tokens = in.rows;
    check_vector(what, "routing.weights", &weights_in, with_last(x_in, k));
    if (weights_in.scalar_type() != at::kFloat) fail(Failure::kValue, "expert_feed_forward: routing.weights must be torch.float32 (got " + name_of(weights_in.scalar_type()) + ")");
    if (tokens > LLSA_MAX_SLOTS / k) fail(Failure::kValue, "expert_feed_forward: too many tokens (" + std::to_string(tokens) + ")");
    const int64_t rows = tokens * k;
    check_ints(what, "routing.experts", experts_in, with_last(x_in, k));
    check_ints(what, "routing.places", places_in, with_last(x_in, k));
    check_ints(what, "routing.order", order_in, {rows});
    check_ints(what, "routing.offsets", offsets_in, {E + 1});
    const bool grad = wants({&x_in, &weights_in, &w1_in, b1, &w2_in, b2, gate_p, residual_p});
    const bool inner = grad && wants({&x_in, &w1_in, b1}), outer = grad && wants({&w2_in, b2}), gates = grad && wants({gate_p}), chooses = grad && wants({&weights_in});
    Tensor out, slopes, h, y, gate, weights, order, offsets, places;
    Rows x;
    Weights w1, w2;
    std::shared_ptr<ExpertFeedForwardBackward> node;
    {
        at::AutoDispatchBelowADInplaceOrView below;
        c10::OptionalDeviceGuard guard(lib->device ? std::optional<at::Device>(x_in.device()) : std::nullopt);
        Call call(*lib, x_in);
        out = at::empty(with_last(x_in, N), x_in.options());
        gate = dense_vector(gate_p);
        order = contiguous(order_in); offsets = contiguous(offsets_in); places = contiguous(places_in); weights = contiguous(weights_in);
        x.t = x_in; w1.rows.t = w1_in; w2.rows.t = w2_in;
        if (tokens > 0) {
            call.operands({{&x_in, &x}, {&w1_in, &w1.rows}, {&w2_in, &w2.rows}});
            w1.E = w2.E = E; w1.N = F; w1.K = pad8(C); w2.N = N; w2.K = pad8(F);
            const Tensor bias1 = dense_bias(b1), bias2 = dense_bias(b2);
            h = call.rows(rows, F);
            if (inner) slopes = slopes_of(call, rows, F);
            y = wide_rows(call, rows, N);
            llsa_experts_args a{};
            a.order = ints(order); a.offsets = ints(offsets); a.places = ints(places);
            a.rows = rows; a.tokens = tokens; a.k = static_cast<int32_t>(k); a.dtype = dtype; a.padded = 1;
            a.E = static_cast<int32_t>(E);
            llsa_experts_args one = a, two = a, all = a;
            set_weights(one, w1);
            // (what a backward wants in the order of the places is brought there once)
            x.cols = C;
            if (grad || !lib->experts_gathers(rows, one.E, one.N, one.K)) x = gathered(call, x, a, nullptr, Tensor(), 1);
            else one.gather_x = 1;
            one.x = x.p(); one.ldx = x.ld;
            one.bias = bias1.defined() ? bias1.data_ptr() : nullptr;
            one.out = h.data_ptr(); one.ldo = h.size(1); one.act = act;
            if (slopes.defined()) { one.slopes = slopes.data_ptr(); one.ldz = slopes.size(1); }
            lib->check(lib->experts_fwd(&one, call.stream()), "experts_fwd");
            set_weights(two, w2);
            two.x = h.data_ptr(); two.ldx = h.size(1); two.bias = bias2.defined() ? bias2.data_ptr() : nullptr;
            two.out = y.data_ptr(); two.ldo = y.size(1); two.wide = 1;
            two.gaps = 1;                                     // (a caller's places may lie where no expert's rows do)
            lib->check(lib->experts_fwd(&two, call.stream()), "experts_fwd");
            const Rows residual = call.addend(residual_p);
            all.weights = weights.data_ptr<float>();
            all.x = y.data_ptr(); all.ldx = y.size(1); all.E = static_cast<int32_t>(E); all.N = static_cast<int32_t>(N); all.K = 8; all.padded = 0;
            if (gate.defined()) { all.gate = gate.data_ptr(); all.s_gate = gate.size(0) > 1 ? gate.stride(0) : 0; }
            all.residual = residual.p(); all.ldr = residual.ld; all.per_sample = in.per_sample();
            all.out = out.data_ptr(); all.ldo = N;
            lib->check(lib->experts_combine(&all, call.stream()), "experts_combine");
        }
        if (grad) {
            node = make_node<ExpertFeedForwardBackward>(lib);
            node->sizes = x_in.sizes().vec(); node->chosen = weights_in.sizes().vec();
            node->tokens = tokens; node->k = k; node->per_sample = in.per_sample(); node->samples = in.samples; node->E = E; node->C = C; node->F = F; node->N = N;
            node->has_b1 = b1 != nullptr; node->has_b2 = b2 != nullptr; node->has_gate = gate_p != nullptr; node->has_residual = residual_p != nullptr;
            node->dtype = dtype;
        }
    }
    if (node) {
        node->set_next_edges(torch::autograd::collect_next_edges(present({&x_in, &weights_in, &w1_in, b1, &w2_in, b2, gate_p, residual_p})));
        torch::autograd::set_history(out, node);
        auto keep = [&](bool needed, const Tensor& t, const Tensor& input) { node->keep(needed ? t : Tensor(), input); };
        const bool any = inner || outer || chooses || gates;
        keep(wants({&w1_in, b1}), x.t, x.t);                  // (in the order of the places)
        keep(x_in.requires_grad(), w1.rows.t, w1_in);
        keep(inner, w2.rows.t, w2_in);
        node->keep(gate, gate_p != nullptr ? *gate_p : gate);
        keep(any, offsets, offsets_in);
        keep(any, order, order_in);
        keep(any, places, places_in);
        keep(any, weights, weights_in);
        keep(inner, slopes, slopes);
        keep(outer, h, h);
        keep(chooses || gates, y, y);
    }
    return out;
}

}  // namespace

void bind_experts(py::module_& m) {
    typedef std::shared_ptr<Library> Lib;
    typedef std::optional<Tensor> Optional;
    m.def("route_tokens", torch::wrap_pybind_function([](const Lib& lib, const Tensor& logits, int64_t k, bool normalize) {
        return without_interpreter([&] { return route_tokens(lib, logits, k, normalize); });
    }));
    m.def("grouped_linear", torch::wrap_pybind_function([](const Lib& lib, const Tensor& x, const Tensor& w, const Tensor& offsets, const Optional& bias, int64_t act) {
        return without_interpreter([&] { return grouped_linear(lib, x, w, offsets, bias, act); });
    }));
    m.def("expert_feed_forward", torch::wrap_pybind_function([](const Lib& lib, const Tensor& x, const Tensor& weights, const Tensor& experts, const Tensor& order, const Tensor& offsets,
                                                                const Tensor& places, const Tensor& w1, const Optional& b1, const Tensor& w2, const Optional& b2, int64_t act,
                                                                const Optional& gate, const Optional& residual) {
        return without_interpreter([&] { return expert_feed_forward(lib, x, weights, experts, order, offsets, places, w1, b1, w2, b2, act, gate, residual); });
    }));
}
