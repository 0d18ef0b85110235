// The operators beside the losses, for torch: layer norm, the causal convolution
// and the selective scan (the latter two also one step at a time), and the rules
// on logits.  Each is differentiable where it has a backward pass; without
// gradients to track it goes straight to the C ABI.  Arguments are checked here
// (RuntimeError through TORCH_CHECK); nothing synchronises with the host.
#include "binding_common.h"

namespace {

using torch::autograd::AutogradContext;
using torch::autograd::tensor_list;
using Maybe = c10::optional<torch::Tensor>;

bool given(const Maybe &t) { return t.has_value() && t->defined(); }

bool is_native(const torch::Tensor &t) {
    return t.scalar_type() == at::ScalarType::Float || t.scalar_type() == at::ScalarType::Half ||
           t.scalar_type() == at::ScalarType::BFloat16;
}

int type_of(const torch::Tensor &t) {
    switch (t.scalar_type()) {
        case at::ScalarType::Half: return WARPCTCT_F16;
        case at::ScalarType::BFloat16: return WARPCTCT_BF16;
        default: return WARPCTCT_F32;
    }
}

// float32, float16 and bfloat16 as they are, any other type as float32 (as the
// losses take their inputs)
torch::Tensor native(const torch::Tensor &t) {
    TORCH_CHECK(!t.is_complex(), "complex tensors are not supported");
    return is_native(t) ? t : t.to(at::ScalarType::Float);
}

void check_on(const torch::Tensor &t, const torch::Tensor &like, const char *name) {
    TORCH_CHECK(t.device() == like.device(), name, " must be located on the same GPU as the input");
}

bool tracked(const torch::Tensor &t) { return t.defined() && t.requires_grad() && at::GradMode::is_enabled(); }
bool tracked(const Maybe &t) { return given(t) && tracked(*t); }

// The gradients are not differentiable themselves: asked for that, a backward
// pass refuses instead of returning them as constants.
void refuse_second_derivative(const char *name) {
    TORCH_CHECK(!at::GradMode::is_enabled(), name, ": the gradient of the gradient is not available "
                "(create_graph=True)");
}

// Nor is there a forward-mode derivative: an input that carries a tangent is
// refused, instead of giving a result without one.
bool has_tangent(const torch::Tensor &t) { return t.defined() && t._fw_grad(0).defined(); }
bool has_tangent(const Maybe &t) { return given(t) && has_tangent(*t); }
template <typename... Inputs>
void refuse_tangents(const char *what, const Inputs &...inputs) {
    if (!c10::AutogradState::get_tls_state().get_fw_grad_mode()) return;
    TORCH_CHECK(!(has_tangent(inputs) || ...), what, ": the forward-mode derivative is not available");
}

const void *ptr(const torch::Tensor &t) { return t.defined() ? t.data_ptr() : nullptr; }
float *floats(const torch::Tensor &t) { return t.defined() ? t.data_ptr<float>() : nullptr; }

// An uninitialised tensor on the device of `like`.  (Below autograd in the
// dispatcher: these calls are a good part of what a step costs the host.)
torch::Tensor fresh(at::IntArrayRef sizes, at::ScalarType type, const torch::Tensor &like) {
    const at::AutoDispatchBelowAutograd below;
    return at::empty(sizes, like.options().dtype(type));
}
torch::Tensor fresh(at::IntArrayRef sizes, const torch::Tensor &like) {
    return fresh(sizes, like.scalar_type(), like);
}
torch::Tensor fresh_bytes(size_t bytes, const torch::Tensor &like) {
    return fresh({static_cast<int64_t>(bytes)}, at::ScalarType::Byte, like);
}
constexpr at::ScalarType kFloat = at::ScalarType::Float;

// ---- layer norm --------------------------------------------------------------

// The rows of a tensor (everything but its last dimension) by two strides; a
// tensor that needs more, or whose last dimension is not dense, is copied.
struct Rows {
    torch::Tensor t;
    long rows = 1, inner = 1, outer_stride = 0, inner_stride = 0;
    explicit Rows(const torch::Tensor &of) : t(of) {
        if (!fits()) {
            t = of.contiguous();
            TORCH_INTERNAL_ASSERT(fits());
        }
    }

   private:
    bool fits() {
        const int64_t last = t.dim() - 1;
        rows = 1;
        for (int64_t d = 0; d < last; ++d) rows *= t.size(d);
        inner = rows > 0 ? rows : 1;
        inner_stride = t.size(last);
        outer_stride = 0;
        if (t.numel() == 0) return true;
        if (t.size(last) > 1 && t.stride(last) != 1) return false;
        int groups = 0;
        int64_t size[2] = {1, 1}, stride[2] = {t.size(last), 0};
        for (int64_t d = last - 1; d >= 0; --d) {
            if (t.size(d) == 1) continue;
            if (groups > 0 && t.stride(d) == size[groups - 1] * stride[groups - 1]) {
                size[groups - 1] *= t.size(d);
            } else {
                if (groups == 2) return false;
                size[groups] = t.size(d);
                stride[groups++] = t.stride(d);
            }
        }
        inner = size[0];
        inner_stride = stride[0];
        outer_stride = stride[1];
        return true;
    }
};

struct NormCall {
    Rows x;
    warpctct_norm_t p;
    NormCall(const torch::Tensor &in, const torch::Tensor &weight, const torch::Tensor &bias, double eps)
        : x(in), p() {
        p.dtype = type_of(x.t);
        p.weight_dtype = weight.defined() ? type_of(weight) : bias.defined() ? type_of(bias) : WARPCTCT_F32;
        p.width = static_cast<int>(in.size(-1));
        p.eps = static_cast<float>(eps);
        p.rows = x.rows;
        p.x_inner_rows = x.inner;
        p.x_outer_stride = x.outer_stride;
        p.x_inner_stride = x.inner_stride;
        p.x = x.t.data_ptr();
        p.weight = ptr(weight);
        p.bias = ptr(bias);
    }
};

// out, and with `keep` what the backward pass needs of every row
std::tuple<torch::Tensor, torch::Tensor> norm_forward(NormCall &call, bool keep) {
    const DeviceGuard guard(device_of(call.x.t));
    auto out = fresh(call.x.t.sizes(), call.x.t);
    torch::Tensor stats;
    if (keep) {
        stats = fresh({call.p.rows, 3}, kFloat, call.x.t);
        call.p.stats = stats.data_ptr<float>();
    }
    call.p.out = out.data_ptr();
    check_rc(warpctct_layer_norm(&call.p, current_stream()), "layer_norm");
    return std::make_tuple(out, stats);
}

class LayerNorm : public torch::autograd::Function<LayerNorm> {
   public:
    static torch::Tensor forward(AutogradContext *ctx, const torch::Tensor &x, const Maybe &weight,
                                 const Maybe &bias, const double eps, const bool track_x,
                                 const bool track_weight, const bool track_bias) {
        const torch::Tensor w = given(weight) ? *weight : torch::Tensor();
        const torch::Tensor b = given(bias) ? *bias : torch::Tensor();
        NormCall call(x, w, b, eps);
        auto out = norm_forward(call, true);
        ctx->save_for_backward({x, w, std::get<1>(out)});
        ctx->saved_data["track"] = std::vector<int64_t>{track_x, track_weight, track_bias};
        ctx->saved_data["weight_dtype"] = static_cast<int64_t>(call.p.weight_dtype);
        return std::get<0>(out);
    }

    static tensor_list backward(AutogradContext *ctx, tensor_list grad_outputs) {
        refuse_second_derivative("layer_norm");
        const auto saved = ctx->get_saved_variables();
        const auto track = ctx->saved_data["track"].toIntVector();
        const torch::Tensor &stats = saved[2];
        NormCall call(saved[0], saved[1], torch::Tensor(), 0.0);
        call.p.weight_dtype = static_cast<int>(ctx->saved_data["weight_dtype"].toInt());
        const torch::Tensor &x = call.x.t;
        const DeviceGuard guard(device_of(x));
        call.p.stats = stats.data_ptr<float>();
        const Rows g(grad_outputs[0]);
        warpctct_norm_grad_t grads = {};
        grads.inner_rows = g.inner;
        grads.outer_stride = g.outer_stride;
        grads.inner_stride = g.inner_stride;
        grads.grad_out = g.t.data_ptr();
        torch::Tensor gx, gw, gb, workspace;
        if (track[0]) gx = fresh(x.sizes(), x);
        const auto params = call.p.weight_dtype == call.p.dtype ? x.scalar_type() : kFloat;
        if (track[1]) gw = fresh({call.p.width}, params, x);
        if (track[2]) gb = fresh({call.p.width}, params, x);
        grads.grad_x = gx.defined() ? gx.data_ptr() : nullptr;
        grads.grad_weight = gw.defined() ? gw.data_ptr() : nullptr;
        grads.grad_bias = gb.defined() ? gb.data_ptr() : nullptr;
        if (track[1] || track[2])
            workspace = fresh_bytes(warpctct_layer_norm_workspace_bytes(call.p.rows, call.p.width), x);
        check_rc(warpctct_layer_norm_grad(&call.p, &grads, workspace.defined() ? workspace.data_ptr() : nullptr,
                                          workspace.defined() ? workspace.numel() : 0, current_stream()),
                 "layer_norm");
        return {gx, gw, gb, torch::Tensor(), torch::Tensor(), torch::Tensor(), torch::Tensor()};
    }
};

torch::Tensor layer_norm(const torch::Tensor &input, Maybe weight, Maybe bias, const double eps) {
    CHECK_DEVICE(input);
    TORCH_CHECK(input.dim() >= 1 && input.size(-1) >= 1, "layer_norm: the input needs a last dimension");
    TORCH_CHECK(input.size(-1) <= (1L << 27) - 32 && input.numel() / input.size(-1) < (1L << 31),
                "layer_norm: at most 2^31 - 1 rows of at most 2^27 - 32 elements");
    TORCH_CHECK(eps >= 0, "layer_norm: eps must not be negative");
    refuse_tangents("layer_norm", input, weight, bias);
    const torch::Tensor x = native(input);
    bool same = true;      // parameters in the input's type; otherwise all of them in float32
    for (const Maybe *p : {&weight, &bias}) {
        if (!given(*p)) continue;
        const char *name = p == &weight ? "weight" : "bias";
        TORCH_CHECK((*p)->dim() == 1 && (*p)->size(0) == x.size(-1), "layer_norm: ", name,
                    " must have one element for each of the input's last dimension");
        check_on(**p, x, name);
        same = same && (*p)->scalar_type() == x.scalar_type();
    }
    for (Maybe *p : {&weight, &bias})
        if (given(*p) && !((same || (*p)->scalar_type() == kFloat) && (*p)->is_contiguous()))
            *p = (same ? **p : native(**p).to(kFloat)).contiguous();
    const bool tx = tracked(x), tw = tracked(weight), tb = tracked(bias);
    if (tx || tw || tb) return LayerNorm::apply(x, weight, bias, eps, tx, tw, tb);
    NormCall call(x, given(weight) ? *weight : torch::Tensor(), given(bias) ? *bias : torch::Tensor(), eps);
    return std::get<0>(norm_forward(call, false));
}

// ---- what the operators along time share ---------------------------------------

int int_size(const torch::Tensor &t, int64_t d, const char *what) {
    TORCH_CHECK(t.size(d) <= 0x7fffffff, what, ": a dimension is too large");
    return static_cast<int>(t.size(d));
}

// a tensor whose last dimension is dense (a copy, if it is not)
torch::Tensor dense_last(const torch::Tensor &t) {
    return t.numel() == 0 || t.size(-1) == 1 || t.stride(-1) == 1 ? t : t.contiguous();
}

// Lengths as int32.  The kernels clamp them into [0, most]; of types that hold
// more than int32 does that has to come before the conversion.
torch::Tensor lengths_of(const Maybe &lengths, const torch::Tensor &x, int64_t most, const char *what) {
    if (!given(lengths)) return torch::Tensor();
    const auto type = lengths->scalar_type();
    TORCH_CHECK(lengths->dim() == 1 && lengths->size(0) == x.size(0) && at::isIntegralType(type, false), what,
                ": lengths must be whole numbers, one for each sequence");
    check_on(*lengths, x, "lengths");
    if (type == at::ScalarType::Long) return as_int32(lengths->clamp(0, most));
    if (type == at::ScalarType::UInt32) return as_int32(lengths->to(at::ScalarType::Long).clamp(0, most));
    if (type == at::ScalarType::UInt64) {      // (from 2^63 on negative as int64)
        const auto wide = lengths->to(at::ScalarType::Long);
        return as_int32(wide.clamp(0, most).masked_fill(wide.lt(0), most));
    }
    return as_int32(*lengths);
}

torch::Tensor flags_of(const Maybe &advance, const torch::Tensor &x, const char *what) {
    if (!given(advance)) return torch::Tensor();
    TORCH_CHECK(advance->dim() == 1 && advance->size(0) == x.size(0) &&
                    advance->scalar_type() == at::ScalarType::Bool,
                what, ": advance must be truth values, one for each sequence");
    check_on(*advance, x, "advance");
    return advance->contiguous();
}

// A step updates its state in place and has no backward pass.  (It counts up the
// state's version first, so that a graph that saved the state refuses to use it.)
void refuse_gradient(std::initializer_list<const Maybe *> inputs, const char *what) {
    for (const Maybe *t : inputs)
        TORCH_CHECK(!tracked(*t), what, ": not differentiable; call it under torch.no_grad()");
}

// ---- causal convolution ----------------------------------------------------------

struct ConvInputs {
    torch::Tensor x, weight, bias, lengths, initial;
    warpctct_conv_t call() const {
        warpctct_conv_t p = {};
        p.dtype = type_of(x);
        p.N = static_cast<int>(x.size(0));
        p.L = static_cast<int>(x.size(1));
        p.E = static_cast<int>(x.size(2));
        p.K = static_cast<int>(weight.size(1));
        p.x_n = x.stride(0);
        p.x_t = x.stride(1);
        p.x = x.data_ptr();
        p.weight = floats(weight);
        p.bias = floats(bias);
        p.lengths = lengths.defined() ? lengths.data_ptr<int>() : nullptr;
        p.initial = ptr(initial);
        return p;
    }
};

tensor_list conv_forward(const ConvInputs &in, bool silu, bool want_state) {
    const DeviceGuard guard(device_of(in.x));
    auto p = in.call();
    p.silu = silu ? 1 : 0;
    tensor_list outs = {fresh(in.x.sizes(), in.x)};
    if (want_state) outs.push_back(fresh({p.N, p.K - 1, p.E}, in.x));
    p.out = outs[0].data_ptr();
    p.last = want_state ? outs[1].data_ptr() : nullptr;
    check_rc(warpctct_causal_conv(&p, current_stream()), "causal_conv");
    return outs;
}

class CausalConv : public torch::autograd::Function<CausalConv> {
   public:
    static tensor_list forward(AutogradContext *ctx, const torch::Tensor &x, const torch::Tensor &weight,
                               const Maybe &bias, const Maybe &initial, const Maybe &lengths, const bool silu,
                               const bool want_state, const bool track_weight, const bool track_bias,
                               const bool track_initial) {
        const auto plain = [](const Maybe &t) { return given(t) ? *t : torch::Tensor(); };
        const ConvInputs in = {x, weight, plain(bias), plain(lengths), plain(initial)};
        ctx->save_for_backward({in.x, in.weight, in.bias, in.lengths, in.initial});
        ctx->saved_data["silu"] = silu;
        ctx->saved_data["track"] = std::vector<int64_t>{track_weight, track_bias, track_initial};
        ctx->set_materialize_grads(false);
        return conv_forward(in, silu, want_state);
    }

    static tensor_list backward(AutogradContext *ctx, tensor_list grad_outputs) {
        refuse_second_derivative("causal_conv");
        const auto saved = ctx->get_saved_variables();
        const ConvInputs in = {saved[0], saved[1], saved[2], saved[3], saved[4]};
        const auto track = ctx->saved_data["track"].toIntVector();
        const DeviceGuard guard(device_of(in.x));
        auto p = in.call();
        p.silu = ctx->saved_data["silu"].toBool() ? 1 : 0;
        const torch::Tensor up = grad_outputs[0].defined() ? dense_last(grad_outputs[0])
                                                           : torch::zeros(in.x.sizes(), in.x.options());
        torch::Tensor glast;
        if (grad_outputs.size() > 1 && grad_outputs[1].defined()) glast = grad_outputs[1].contiguous();
        torch::Tensor gx = fresh(in.x.sizes(), in.x), gw, gb, ginitial, workspace;
        if (track[0]) gw = fresh({p.E, p.K}, kFloat, in.x);
        if (track[1]) gb = fresh({p.E}, kFloat, in.x);
        if (track[2]) ginitial = fresh(in.initial.sizes(), in.x);
        if (track[0] || track[1])
            workspace = fresh_bytes(warpctct_causal_conv_workspace_bytes(p.N, p.L, p.E, p.K), in.x);
        warpctct_conv_grad_t g = {};
        g.grad_n = up.stride(0);
        g.grad_t = up.stride(1);
        g.grad_out = up.data_ptr();
        g.grad_last = ptr(glast);
        g.grad_x = gx.data_ptr();
        g.grad_initial = ginitial.defined() ? ginitial.data_ptr() : nullptr;
        g.grad_weight = floats(gw);
        g.grad_bias = floats(gb);
        check_rc(warpctct_causal_conv_grad(&p, &g, workspace.defined() ? workspace.data_ptr() : nullptr,
                                           workspace.defined() ? workspace.numel() : 0, current_stream()),
                 "causal_conv");
        return {gx, gw, gb, ginitial, torch::Tensor(), torch::Tensor(), torch::Tensor(), torch::Tensor(),
                torch::Tensor(), torch::Tensor()};
    }
};

// weight (E, K) and bias (E), in float32
void check_taps(const torch::Tensor &weight, const Maybe &bias, const torch::Tensor &x, const char *what) {
    TORCH_CHECK(weight.dim() == 2 && weight.size(0) == x.size(-1) && weight.size(1) >= 1 &&
                    weight.size(1) <= WARPCTCT_CONV_MAX_TAPS,
                what, ": weight must be (channels, taps) with 1 to ", static_cast<int>(WARPCTCT_CONV_MAX_TAPS),
                " taps");
    check_on(weight, x, "weight");
    if (!given(bias)) return;
    TORCH_CHECK(bias->dim() == 1 && bias->size(0) == x.size(-1), what, ": bias must have one element a channel");
    check_on(*bias, x, "bias");
}
torch::Tensor as_float(const torch::Tensor &t) {
    TORCH_CHECK(!t.is_complex(), "complex tensors are not supported");
    return t.scalar_type() == kFloat && t.is_contiguous() ? t : t.to(kFloat).contiguous();
}

tensor_list causal_conv(const torch::Tensor &input, const torch::Tensor &weight, const Maybe &bias,
                        const Maybe &lengths, const Maybe &initial, const bool silu, const bool want_state) {
    CHECK_DEVICE(input);
    TORCH_CHECK(input.dim() == 3 && input.size(2) >= 1, "causal_conv: the input must be (batch, time, channels)");
    refuse_tangents("causal_conv", input, weight, bias, initial);
    const torch::Tensor x = dense_last(native(input));
    check_taps(weight, bias, x, "causal_conv");
    const int L = int_size(x, 1, "causal_conv"), E = int_size(x, 2, "causal_conv");
    TORCH_CHECK(x.size(0) <= 65535 && L <= (1L << 30) && static_cast<long>(L) * E <= (1L << 32) - 1024,
                "causal_conv: at most 65535 sequences of at most 2^30 steps and 2^32 - 1024 elements");
    ConvInputs in = {x, as_float(weight), given(bias) ? as_float(*bias) : torch::Tensor(),
                     lengths_of(lengths, x, L, "causal_conv"), torch::Tensor()};
    if (given(initial)) {
        const torch::Tensor first = native(*initial);
        TORCH_CHECK(first.dim() == 3 && first.size(0) == x.size(0) && first.size(1) == weight.size(1) - 1 &&
                        first.size(2) == E && first.scalar_type() == x.scalar_type(),
                    "causal_conv: initial_state must be (batch, taps - 1, channels) in the input's type");
        check_on(first, x, "initial_state");
        in.initial = first.contiguous();
    }
    const bool tw = tracked(in.weight), tb = tracked(in.bias), ti = tracked(in.initial);
    if (!(tracked(in.x) || tw || tb || ti)) return conv_forward(in, silu, want_state);
    const auto maybe = [](const torch::Tensor &t) { return t.defined() ? Maybe(t) : Maybe(); };
    return CausalConv::apply(in.x, in.weight, maybe(in.bias), maybe(in.initial), maybe(in.lengths), silu, want_state,
                             tw, tb, ti);
}

torch::Tensor causal_conv_step(const torch::Tensor &input, torch::Tensor state, const torch::Tensor &weight,
                               const Maybe &bias, const bool silu, const Maybe &advance) {
    CHECK_DEVICE(input);
    TORCH_CHECK(input.dim() == 2 && input.size(1) >= 1, "causal_conv_step: the input must be (batch, channels)");
    refuse_tangents("causal_conv_step", input, state, weight, bias);
    const torch::Tensor x = dense_last(native(input));
    check_taps(weight, bias, x, "causal_conv_step");
    const Maybe all[4] = {x, state, weight, bias};
    refuse_gradient({&all[0], &all[1], &all[2], &all[3]}, "causal_conv_step");
    TORCH_CHECK(state.dim() == 3 && state.size(0) == x.size(0) && state.size(1) == weight.size(1) - 1 &&
                    state.size(2) == x.size(1) && state.scalar_type() == x.scalar_type() && state.is_contiguous(),
                "causal_conv_step: state must be (batch, taps - 1, channels), dense, in the input's type");
    check_on(state, x, "state");
    const torch::Tensor go = flags_of(advance, x, "causal_conv_step");
    const torch::Tensor w = as_float(weight), b = given(bias) ? as_float(*bias) : torch::Tensor();
    const DeviceGuard guard(device_of(x));
    torch::autograd::impl::bump_version(state);
    auto out = fresh(x.sizes(), x);
    warpctct_conv_step_t p = {};
    p.dtype = type_of(x);
    p.N = int_size(x, 0, "causal_conv_step");
    p.E = int_size(x, 1, "causal_conv_step");
    p.K = static_cast<int>(weight.size(1));
    p.silu = silu ? 1 : 0;
    p.x_n = x.stride(0);
    p.x = x.data_ptr();
    p.state = state.data_ptr();
    p.weight = floats(w);
    p.bias = floats(b);
    p.advance = go.defined() ? reinterpret_cast<const unsigned char *>(go.data_ptr<bool>()) : nullptr;
    p.out = out.data_ptr();
    check_rc(warpctct_causal_conv_step(&p, current_stream()), "causal_conv_step");
    return out;
}

// ---- selective scan ----------------------------------------------------------------

struct ScanInputs {
    torch::Tensor x, dt, a, b, c, skip, gate, dt_bias, lengths, initial;
    warpctct_scan_t call() const {
        warpctct_scan_t p = {};
        p.dtype = type_of(x);
        p.N = static_cast<int>(x.size(0));
        p.L = static_cast<int>(x.size(1));
        p.E = static_cast<int>(x.size(2));
        p.S = static_cast<int>(a.size(1));
        p.G = static_cast<int>(b.size(2));
        p.x_n = x.stride(0);
        p.x_t = x.stride(1);
        p.dt_n = dt.stride(0);
        p.dt_t = dt.stride(1);
        if (gate.defined()) {
            p.gate_n = gate.stride(0);
            p.gate_t = gate.stride(1);
        }
        p.b_n = b.stride(0);
        p.b_t = b.stride(1);
        p.b_g = b.stride(2);
        p.c_n = c.stride(0);
        p.c_t = c.stride(1);
        p.c_g = c.stride(2);
        p.x = x.data_ptr();
        p.dt = dt.data_ptr();
        p.gate = ptr(gate);
        p.b = b.data_ptr();
        p.c = c.data_ptr();
        p.a = floats(a);
        p.skip = floats(skip);
        p.dt_bias = floats(dt_bias);
        p.lengths = lengths.defined() ? lengths.data_ptr<int>() : nullptr;
        p.initial = floats(initial);
        return p;
    }
};

// out, the last states if wanted, and what the backward pass needs
std::tuple<tensor_list, torch::Tensor> scan_forward(const ScanInputs &in, bool softplus, bool want_state,
                                                    bool for_backward) {
    const DeviceGuard guard(device_of(in.x));
    auto p = in.call();
    p.softplus = softplus ? 1 : 0;
    tensor_list outs = {fresh(in.x.sizes(), in.x)};
    if (want_state)
        outs.push_back(fresh({p.N, p.E, p.S}, kFloat, in.x));
    p.out = outs[0].data_ptr();
    p.last = want_state ? floats(outs[1]) : nullptr;
    torch::Tensor keep;
    if (for_backward) keep = fresh_bytes(warpctct_selective_scan_keep_bytes(p.N, p.L, p.E, p.S), in.x);
    const size_t scratch = warpctct_selective_scan_workspace_bytes(p.N, p.L, p.E, p.S, p.G, 0);
    torch::Tensor workspace;
    if (scratch > 0) workspace = fresh_bytes(scratch, in.x);
    check_rc(warpctct_selective_scan(&p, keep.defined() ? keep.data_ptr() : nullptr, keep.defined() ? keep.numel() : 0,
                                     workspace.defined() ? workspace.data_ptr() : nullptr, scratch, current_stream()),
             "selective_scan");
    return std::make_tuple(outs, keep);
}

class SelectiveScan : public torch::autograd::Function<SelectiveScan> {
   public:
    static tensor_list forward(AutogradContext *ctx, const torch::Tensor &x, const torch::Tensor &dt,
                               const torch::Tensor &a, const torch::Tensor &b, const torch::Tensor &c,
                               const Maybe &skip, const Maybe &gate, const Maybe &dt_bias, const Maybe &initial,
                               const Maybe &lengths, const bool softplus, const bool want_state,
                               const bool track_initial) {
        const auto plain = [](const Maybe &t) { return given(t) ? *t : torch::Tensor(); };
        const ScanInputs in = {x, dt, a, b, c, plain(skip), plain(gate), plain(dt_bias), plain(lengths),
                               plain(initial)};
        auto got = scan_forward(in, softplus, want_state, true);
        ctx->save_for_backward({in.x, in.dt, in.a, in.b, in.c, in.skip, in.gate, in.dt_bias, in.lengths, in.initial,
                                std::get<1>(got)});
        ctx->saved_data["softplus"] = softplus;
        ctx->saved_data["track_initial"] = track_initial;
        ctx->set_materialize_grads(false);
        return std::get<0>(got);
    }

    static tensor_list backward(AutogradContext *ctx, tensor_list grad_outputs) {
        refuse_second_derivative("selective_scan");
        const auto s = ctx->get_saved_variables();
        const ScanInputs in = {s[0], s[1], s[2], s[3], s[4], s[5], s[6], s[7], s[8], s[9]};
        const torch::Tensor &x = in.x, &keep = s[10];
        const DeviceGuard guard(device_of(x));
        auto p = in.call();
        p.softplus = ctx->saved_data["softplus"].toBool() ? 1 : 0;
        const torch::Tensor up =
            grad_outputs[0].defined() ? dense_last(grad_outputs[0]) : torch::zeros(x.sizes(), x.options());
        torch::Tensor glast;
        if (grad_outputs.size() > 1 && grad_outputs[1].defined()) glast = grad_outputs[1].contiguous();
        torch::Tensor gx = fresh(x.sizes(), x), gdt = fresh(x.sizes(), x), gb = fresh(in.b.sizes(), x),
                      gc = fresh(in.c.sizes(), x), ga = fresh({p.E, p.S}, kFloat, x), gz, gskip, gbias, ginitial;
        if (in.gate.defined()) gz = fresh(x.sizes(), x);
        if (in.skip.defined()) gskip = fresh({p.E}, kFloat, x);
        if (in.dt_bias.defined()) gbias = fresh({p.E}, kFloat, x);
        if (ctx->saved_data["track_initial"].toBool()) ginitial = fresh({p.N, p.E, p.S}, kFloat, x);
        const auto workspace =
            fresh_bytes(warpctct_selective_scan_workspace_bytes(p.N, p.L, p.E, p.S, p.G, 1), x);
        warpctct_scan_grad_t g = {};
        g.grad_n = up.stride(0);
        g.grad_t = up.stride(1);
        g.grad_out = up.data_ptr();
        g.grad_last = floats(glast);
        g.grad_x = gx.data_ptr();
        g.grad_dt = gdt.data_ptr();
        g.grad_gate = gz.defined() ? gz.data_ptr() : nullptr;
        g.grad_b = gb.data_ptr();
        g.grad_c = gc.data_ptr();
        g.grad_a = floats(ga);
        g.grad_skip = floats(gskip);
        g.grad_dt_bias = floats(gbias);
        g.grad_initial = floats(ginitial);
        check_rc(warpctct_selective_scan_grad(&p, &g, keep.data_ptr(), keep.numel(), workspace.data_ptr(),
                                              workspace.numel(), current_stream()),
                 "selective_scan");
        return {gx, gdt, ga, gb, gc, gskip, gz, gbias, ginitial, torch::Tensor(), torch::Tensor(), torch::Tensor(),
                torch::Tensor()};
    }
};

// b or c: (..., S) shared by all channels, or (..., G, S)
torch::Tensor groups_of(const torch::Tensor &t, const torch::Tensor &x, int64_t S, const char *name,
                        const char *what) {
    const int64_t lead = x.dim() - 1;
    TORCH_CHECK(t.dim() == lead + 1 || t.dim() == lead + 2, what, ": ", name, " has the wrong number of dimensions");
    auto v = native(t);
    if (v.dim() == lead + 1) v = v.unsqueeze(lead);
    for (int64_t d = 0; d < lead; ++d)
        TORCH_CHECK(v.size(d) == x.size(d), what, ": ", name, " must have the input's batch and time");
    TORCH_CHECK(v.size(lead) >= 1 && x.size(-1) % v.size(lead) == 0 && v.size(-1) == S, what, ": ", name,
                " must be (..., groups, states), the channels a multiple of the groups");
    TORCH_CHECK(v.scalar_type() == x.scalar_type(), what, ": ", name, " must have the input's type");
    check_on(v, x, name);
    return dense_last(v);
}

torch::Tensor like_input(const torch::Tensor &t, const torch::Tensor &x, const char *name, const char *what) {
    const auto v = native(t);
    TORCH_CHECK(v.sizes() == x.sizes() && v.scalar_type() == x.scalar_type(), what, ": ", name,
                " must have the input's shape and type");
    check_on(v, x, name);
    return dense_last(v);
}

torch::Tensor per_channel(const Maybe &t, const torch::Tensor &x, const char *name, const char *what) {
    if (!given(t)) return torch::Tensor();
    TORCH_CHECK(t->dim() == 1 && t->size(0) == x.size(-1), what, ": ", name, " must have one element a channel");
    check_on(*t, x, name);
    return as_float(*t);
}

// x, dt, a, b, c, skip, gate, dt_bias, checked and in the types of the C ABI
ScanInputs scan_inputs(const torch::Tensor &input, const torch::Tensor &dt, const torch::Tensor &a,
                       const torch::Tensor &b, const torch::Tensor &c, const Maybe &skip, const Maybe &gate,
                       const Maybe &dt_bias, const char *what) {
    ScanInputs in;
    in.x = dense_last(native(input));
    TORCH_CHECK(a.dim() == 2 && a.size(0) == in.x.size(-1) && a.size(1) >= 1 &&
                    a.size(1) <= WARPCTCT_SCAN_MAX_STATES,
                what, ": a must be (channels, states) with 1 to ", static_cast<int>(WARPCTCT_SCAN_MAX_STATES),
                " states");
    check_on(a, in.x, "a");
    TORCH_CHECK(in.x.size(-1) < (1 << 24), what, ": fewer than 2^24 channels");
    in.a = as_float(a);
    in.dt = like_input(dt, in.x, "dt", what);
    in.b = groups_of(b, in.x, a.size(1), "b", what);
    in.c = groups_of(c, in.x, a.size(1), "c", what);
    TORCH_CHECK(in.b.sizes() == in.c.sizes(), what, ": b and c must have the same groups");
    in.skip = per_channel(skip, in.x, "skip", what);
    in.dt_bias = per_channel(dt_bias, in.x, "dt_bias", what);
    if (given(gate)) in.gate = like_input(*gate, in.x, "gate", what);
    return in;
}

tensor_list selective_scan(const torch::Tensor &input, const torch::Tensor &dt, const torch::Tensor &a,
                           const torch::Tensor &b, const torch::Tensor &c, const Maybe &skip, const Maybe &gate,
                           const Maybe &dt_bias, const bool softplus, const Maybe &lengths, const Maybe &initial,
                           const bool want_state) {
    const char *what = "selective_scan";
    CHECK_DEVICE(input);
    TORCH_CHECK(input.dim() == 3 && input.size(2) >= 1, "selective_scan: the input must be (batch, time, channels)");
    TORCH_CHECK(input.size(0) <= 65535 && input.size(1) < (1L << 30),
                "selective_scan: at most 65535 sequences of fewer than 2^30 steps");
    refuse_tangents(what, input, dt, a, b, c, skip, gate, dt_bias, initial);
    ScanInputs in = scan_inputs(input, dt, a, b, c, skip, gate, dt_bias, what);
    in.lengths = lengths_of(lengths, in.x, in.x.size(1), what);
    if (given(initial)) {
        const torch::Tensor first = native(*initial);
        TORCH_CHECK(first.dim() == 3 && first.size(0) == in.x.size(0) && first.size(1) == in.x.size(2) &&
                        first.size(2) == a.size(1) && first.scalar_type() == kFloat,
                    "selective_scan: initial_state must be (batch, channels, states) in float32");
        check_on(first, in.x, "initial_state");
        in.initial = first.contiguous();
    }
    bool track = false;
    for (const auto *t : {&in.x, &in.dt, &in.a, &in.b, &in.c, &in.skip, &in.gate, &in.dt_bias, &in.initial})
        track = track || tracked(*t);
    if (!track) return std::get<0>(scan_forward(in, softplus, want_state, false));
    const auto maybe = [](const torch::Tensor &t) { return t.defined() ? Maybe(t) : Maybe(); };
    return SelectiveScan::apply(in.x, in.dt, in.a, in.b, in.c, maybe(in.skip), maybe(in.gate), maybe(in.dt_bias),
                                maybe(in.initial), maybe(in.lengths), softplus, want_state, tracked(in.initial));
}

torch::Tensor selective_scan_step(const torch::Tensor &input, torch::Tensor state, const torch::Tensor &dt,
                                  const torch::Tensor &a, const torch::Tensor &b, const torch::Tensor &c,
                                  const Maybe &skip, const Maybe &gate, const Maybe &dt_bias, const bool softplus,
                                  const Maybe &advance) {
    const char *what = "selective_scan_step";
    CHECK_DEVICE(input);
    TORCH_CHECK(input.dim() == 2 && input.size(1) >= 1, "selective_scan_step: the input must be (batch, channels)");
    const Maybe all[6] = {input, state, dt, a, b, c};
    refuse_gradient({&all[0], &all[1], &all[2], &all[3], &all[4], &all[5], &skip, &gate, &dt_bias}, what);
    refuse_tangents(what, input, state, dt, a, b, c, skip, gate, dt_bias);
    const ScanInputs in = scan_inputs(input, dt, a, b, c, skip, gate, dt_bias, what);
    const torch::Tensor &x = in.x;
    TORCH_CHECK(state.dim() == 3 && state.size(0) == x.size(0) && state.size(1) == x.size(1) &&
                    state.size(2) == a.size(1) && state.scalar_type() == at::ScalarType::Float &&
                    state.is_contiguous(),
                "selective_scan_step: state must be (batch, channels, states), dense, in float32");
    check_on(state, x, "state");
    const torch::Tensor go = flags_of(advance, x, what);
    const DeviceGuard guard(device_of(x));
    torch::autograd::impl::bump_version(state);
    auto out = fresh(x.sizes(), x);
    warpctct_scan_step_t p = {};
    p.dtype = type_of(x);
    p.N = int_size(x, 0, what);
    p.E = int_size(x, 1, what);
    p.S = static_cast<int>(a.size(1));
    p.G = static_cast<int>(in.b.size(1));
    p.softplus = softplus ? 1 : 0;
    p.x_n = x.stride(0);
    p.dt_n = in.dt.stride(0);
    p.gate_n = in.gate.defined() ? in.gate.stride(0) : 0;
    p.b_n = in.b.stride(0);
    p.b_g = in.b.stride(1);
    p.c_n = in.c.stride(0);
    p.c_g = in.c.stride(1);
    p.x = x.data_ptr();
    p.dt = in.dt.data_ptr();
    p.gate = ptr(in.gate);
    p.b = in.b.data_ptr();
    p.c = in.c.data_ptr();
    p.a = floats(in.a);
    p.skip = floats(in.skip);
    p.dt_bias = floats(in.dt_bias);
    p.state = floats(state);
    p.advance = go.defined() ? reinterpret_cast<const unsigned char *>(go.data_ptr<bool>()) : nullptr;
    p.out = out.data_ptr();
    check_rc(warpctct_selective_scan_step(&p, current_stream()), what);
    return out;
}

// ---- rules on logits ---------------------------------------------------------------

// a penalty: one number for all rows, or a tensor with one for each
struct Penalty {
    float all = 0.0f;
    torch::Tensor each;
    Penalty(const pybind11::object &given, const torch::Tensor &logits, const char *name) {
        if (!THPVariable_Check(given.ptr())) {
            all = given.cast<float>();
            return;
        }
        const auto t = given.cast<torch::Tensor>();
        TORCH_CHECK(t.dim() == 1 && t.size(0) == logits.size(0), "adjust_logits: ", name,
                    " must be a number or one for each row");
        check_on(t, logits, name);
        refuse_if_tracked(t, name);
        each = as_float(t);
    }
    static void refuse_if_tracked(const torch::Tensor &t, const char *name) {
        TORCH_CHECK(!tracked(t), "adjust_logits: not differentiable (", name, "); call it under torch.no_grad()");
        refuse_tangents("adjust_logits", t);
    }
};

torch::Tensor adjust_logits(const torch::Tensor &input, const Maybe &tokens, const Maybe &tokens_lengths,
                            const pybind11::object &repetition, const pybind11::object &presence,
                            const pybind11::object &frequency, const Maybe &bias, const Maybe &allowed) {
    CHECK_DEVICE(input);
    TORCH_CHECK(input.dim() == 2 && input.size(1) >= 1 && input.size(1) <= (1L << 30) && input.size(0) <= 65535,
                "adjust_logits: the logits must be (rows, vocabulary), at most 65535 rows of at most 2^30");
    Penalty::refuse_if_tracked(input, "logits");
    const torch::Tensor x = dense_last(native(input));
    const int64_t N = x.size(0), V = x.size(1);
    warpctct_adjust_t p = {};
    p.dtype = type_of(x);
    p.N = static_cast<int>(N);
    p.V = static_cast<int>(V);
    p.logits_n = x.stride(0);
    p.logits = x.data_ptr();
    const Penalty rep(repetition, x, "repetition_penalty"), pre(presence, x, "presence_penalty"),
        fre(frequency, x, "frequency_penalty");
    TORCH_CHECK(rep.each.defined() || rep.all > 0.0f, "adjust_logits: repetition_penalty must be positive");
    p.repetition = rep.all;
    p.presence = pre.all;
    p.frequency = fre.all;
    p.repetitions = floats(rep.each);
    p.presences = floats(pre.each);
    p.frequencies = floats(fre.each);
    torch::Tensor history, lengths, b, mask;
    if (given(tokens)) {
        const auto type = tokens->scalar_type();
        TORCH_CHECK(tokens->dim() == 2 && tokens->size(0) == N && at::isIntegralType(type, false) &&
                        tokens->size(1) <= (1L << 30),
                    "adjust_logits: tokens must be whole numbers, (rows, history), a history of at most 2^30");
        check_on(*tokens, x, "tokens");
        // (as int64 what int32 does not hold stays outside the vocabulary)
        const bool taken = type == at::ScalarType::Int || type == at::ScalarType::Long;
        const bool wide = type == at::ScalarType::UInt32 || type == at::ScalarType::UInt64;
        history = dense_last(taken ? *tokens : tokens->to(wide ? at::ScalarType::Long : at::ScalarType::Int));
        p.H = static_cast<int>(history.size(1));
        p.tokens_64 = history.scalar_type() == at::ScalarType::Long ? 1 : 0;
        p.tokens_n = history.stride(0);
        p.tokens = history.data_ptr();
        if (given(tokens_lengths)) {
            lengths = lengths_of(tokens_lengths, x, p.H, "adjust_logits");
            p.tokens_lengths = lengths.data_ptr<int>();
        }
    } else {
        TORCH_CHECK(!given(tokens_lengths), "adjust_logits: tokens_lengths without tokens");
    }
    const auto rows_of = [&](const torch::Tensor &t, int64_t width, const char *name) {
        TORCH_CHECK((t.dim() == 1 || (t.dim() == 2 && t.size(0) == N)) && t.size(-1) == width, "adjust_logits: ",
                    name, " must have ", width, " columns, for all rows or for each");
        check_on(t, x, name);
        return dense_last(t);
    };
    if (given(bias)) {
        Penalty::refuse_if_tracked(*bias, "bias");
        b = rows_of(native(*bias), V, "bias");
        p.bias_dtype = type_of(b);
        p.bias_n = b.dim() == 2 ? b.stride(0) : 0;
        p.bias = b.data_ptr();
    }
    if (given(allowed)) {
        const bool packed = allowed->scalar_type() == at::ScalarType::Int;
        TORCH_CHECK(packed || allowed->scalar_type() == at::ScalarType::Bool,
                    "adjust_logits: allowed must be truth values, or int32 words of 32 bits each");
        mask = rows_of(*allowed, packed ? (V + 31) / 32 : V, "allowed");
        p.allowed_packed = packed ? 1 : 0;
        p.allowed_n = mask.dim() == 2 ? mask.stride(0) : 0;
        p.allowed = mask.data_ptr();
    }
    const DeviceGuard guard(device_of(x));
    auto out = fresh(x.sizes(), x);
    p.out = out.data_ptr();
    check_rc(warpctct_adjust_logits(&p, current_stream()), "adjust_logits");
    return out;
}

}  // namespace

void define_network(pybind11::module &m) {
    m.def("layer_norm", &layer_norm, "Layer norm over the last dimension, differentiable.",
          pybind11::arg("x"), pybind11::arg("weight") = pybind11::none(),
          pybind11::arg("bias") = pybind11::none(), pybind11::arg("eps") = 1e-5);
    m.def("causal_conv", &causal_conv, "Short causal convolution along time, differentiable.",
          pybind11::arg("x"), pybind11::arg("weight"), pybind11::arg("bias"), pybind11::arg("lengths"),
          pybind11::arg("initial_state"), pybind11::arg("silu"), pybind11::arg("return_state"));
    m.def("causal_conv_step", &causal_conv_step, "One step of causal_conv; updates the state in place.",
          pybind11::arg("x"), pybind11::arg("state"), pybind11::arg("weight"), pybind11::arg("bias"),
          pybind11::arg("silu"), pybind11::arg("advance"));
    m.def("adjust_logits", &adjust_logits, "Penalties, biases and masks on logits.", pybind11::arg("logits"),
          pybind11::arg("tokens"), pybind11::arg("tokens_lengths"), pybind11::arg("repetition_penalty"),
          pybind11::arg("presence_penalty"), pybind11::arg("frequency_penalty"), pybind11::arg("bias"),
          pybind11::arg("allowed"));
    m.def("selective_scan", &selective_scan, "Selective state space scan, differentiable.", pybind11::arg("x"),
          pybind11::arg("dt"), pybind11::arg("a"), pybind11::arg("b"), pybind11::arg("c"), pybind11::arg("skip"),
          pybind11::arg("gate"), pybind11::arg("dt_bias"), pybind11::arg("softplus"), pybind11::arg("lengths"),
          pybind11::arg("initial_state"), pybind11::arg("return_state"));
    m.def("selective_scan_step", &selective_scan_step, "One step of selective_scan; updates the state in place.",
          pybind11::arg("x"), pybind11::arg("state"), pybind11::arg("dt"), pybind11::arg("a"), pybind11::arg("b"),
          pybind11::arg("c"), pybind11::arg("skip"), pybind11::arg("gate"), pybind11::arg("dt_bias"),
          pybind11::arg("softplus"), pybind11::arg("advance"));
}
