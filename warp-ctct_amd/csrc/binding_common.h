// What the sources of the torch binding `warp_ctct._C` share: argument checks,
// the current stream, and the element types of the C ABI.
#pragma once

#include <torch/extension.h>

// PyTorch-ROCm presents HIP devices under the "cuda" device type; these are
// its guard and stream accessors for that arrangement.
#include <ATen/hip/impl/HIPGuardImplMasqueradingAsCUDA.h>
#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>

#include <tuple>

#include "warp_ctct_hip.h"

#define CHECK_CONTIGUOUS(x) TORCH_CHECK((x).is_contiguous(), #x " must be contiguous")
#define CHECK_DEVICE(x) TORCH_CHECK((x).device().is_cuda(), #x " must be located on the GPU")
#define CHECK_FLOAT(x) \
    TORCH_CHECK((x).scalar_type() == at::ScalarType::Float, #x " must be a Float tensor")
#define CHECK_INT(x) \
    TORCH_CHECK((x).scalar_type() == at::ScalarType::Int, #x " must be a Int tensor")

inline void check_rc(int rc, const char *what) {
    TORCH_CHECK(rc == WARPCTCT_OK, what, ": ", warpctct_error_string(rc));
}

using DeviceGuard = c10::hip::OptionalHIPGuardMasqueradingAsCUDA;

inline void *current_stream() {
    return static_cast<void *>(c10::hip::getCurrentHIPStreamMasqueradingAsCUDA().stream());
}

// labels and lengths as contiguous int32 (the reference casts with .int(),
// warp_ctct/__init__.py:135-136); tensors that already are cost nothing
inline torch::Tensor as_int32(const torch::Tensor &t) {
    if (t.scalar_type() == at::ScalarType::Int && t.is_contiguous()) return t;
    return t.to(at::ScalarType::Int).contiguous();
}

// The operators beside the losses (binding_network.cpp).
void define_network(pybind11::module &m);
