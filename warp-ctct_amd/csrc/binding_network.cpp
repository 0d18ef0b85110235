// The operators beside the losses, for torch: layer norm.  Each is differentiable where it has a backward pass; without gradients to
// track it goes straight to the C ABI.  Arguments are checked here (RuntimeError
// through TORCH_CHECK); nothing synchronises with the host.
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
torch::Tensor native(const torch::Tensor &t) { return is_native(t) ? t : t.to(at::ScalarType::Float); }

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

const void *ptr(const torch::Tensor &t) { return t.defined() ? t.data_ptr() : nullptr; }
float *floats(const torch::Tensor &t) { return t.defined() ? t.data_ptr<float>() : nullptr; }

torch::Tensor bytes_like(const torch::Tensor &like, size_t bytes) {
    return torch::empty({static_cast<int64_t>(bytes)}, like.options().dtype(at::ScalarType::Byte));
}

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
    auto out = torch::empty(call.x.t.sizes(), call.x.t.options());
    torch::Tensor stats;
    if (keep) {
        stats = torch::empty({call.p.rows, 3}, call.x.t.options().dtype(at::ScalarType::Float));
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
        if (track[0]) gx = torch::empty(x.sizes(), x.options());
        const auto params = x.options().dtype(call.p.weight_dtype == call.p.dtype ? x.scalar_type()
                                                                                  : at::ScalarType::Float);
        if (track[1]) gw = torch::empty({call.p.width}, params);
        if (track[2]) gb = torch::empty({call.p.width}, params);
        grads.grad_x = gx.defined() ? gx.data_ptr() : nullptr;
        grads.grad_weight = gw.defined() ? gw.data_ptr() : nullptr;
        grads.grad_bias = gb.defined() ? gb.data_ptr() : nullptr;
        if (track[1] || track[2])
            workspace = bytes_like(x, warpctct_layer_norm_workspace_bytes(call.p.rows, call.p.width));
        check_rc(warpctct_layer_norm_grad(&call.p, &grads, workspace.defined() ? workspace.data_ptr() : nullptr,
                                          workspace.defined() ? workspace.numel() : 0, current_stream()),
                 "layer_norm");
        return {gx, gw, gb, torch::Tensor(), torch::Tensor(), torch::Tensor(), torch::Tensor()};
    }
};

torch::Tensor layer_norm(const torch::Tensor &input, Maybe weight, Maybe bias, const double eps) {
    CHECK_DEVICE(input);
    TORCH_CHECK(input.dim() >= 1 && input.size(-1) >= 1, "layer_norm: the input needs a last dimension");
    TORCH_CHECK(input.size(-1) < (1L << 30) && input.numel() / input.size(-1) < (1L << 31),
                "layer_norm: at most 2^31 - 1 rows of fewer than 2^30 elements");
    TORCH_CHECK(eps >= 0, "layer_norm: eps must not be negative");
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
        if (given(*p)) *p = (same ? **p : (*p)->to(at::ScalarType::Float)).contiguous();
    const bool tx = tracked(x), tw = tracked(weight), tb = tracked(bias);
    if (tx || tw || tb) return LayerNorm::apply(x, weight, bias, eps, tx, tw, tb);
    NormCall call(x, given(weight) ? *weight : torch::Tensor(), given(bias) ? *bias : torch::Tensor(), eps);
    return std::get<0>(norm_forward(call, false));
}

}  // namespace

void define_network(pybind11::module &m) {
    m.def("layer_norm", &layer_norm, "Layer norm over the last dimension, differentiable.",
          pybind11::arg("x"), pybind11::arg("weight") = pybind11::none(),
          pybind11::arg("bias") = pybind11::none(), pybind11::arg("eps") = 1e-5);
}
