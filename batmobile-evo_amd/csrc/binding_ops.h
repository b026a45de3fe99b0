// Host helpers that the bindings of the transformer operators share: checks of arguments, streams,
// memory, autograd.
#pragma once

#include <c10/core/AutogradState.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/extension.h>

#include "batmobile_hip.h"

namespace bmops {

using torch::Tensor;
using OptTensor = c10::optional<Tensor>;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

inline hipStream_t stream_of(const Tensor& t) {
    return c10::hip::getCurrentHIPStream(t.device().index()).stream();
}

inline void check_status(int rc, const char* what) {
    if (rc == BATMOBILE_HIP_OK) return;
    if (rc == BATMOBILE_HIP_ERR_ARG) TORCH_CHECK(false, what, ": invalid argument");
    if (rc == BATMOBILE_HIP_ERR_WORKSPACE) TORCH_CHECK(false, what, ": workspace too small");
    TORCH_CHECK(false, "HIP error in ", what, ": ", hipGetErrorString(static_cast<hipError_t>(rc)));
}

// 0 fp32, 1 bf16
inline int dtype_of(const Tensor& t, const char* name) {
    TORCH_CHECK(t.is_cuda(), name, " must be a CUDA tensor");
    TORCH_CHECK(t.scalar_type() == torch::kFloat32 || t.scalar_type() == torch::kBFloat16, name,
                " must be float32 or bfloat16");
    return t.scalar_type() == torch::kBFloat16;
}
inline void check_like(const Tensor& t, const Tensor& as, const char* name) {
    TORCH_CHECK(t.device() == as.device(), name, " must be on ", as.device());
    TORCH_CHECK(t.scalar_type() == as.scalar_type(), name, " must have the type of the others");
}
inline void check_f32(const Tensor& t, const Tensor& as, const char* name) {
    TORCH_CHECK(t.device() == as.device(), name, " must be on ", as.device());
    TORCH_CHECK(t.scalar_type() == torch::kFloat32, name, " must be float32");
}
inline void check_same(const Tensor& t, const Tensor& x, const char* name) {
    check_like(t, x, name);
    TORCH_CHECK(t.sizes() == x.sizes(), name, " must have the shape of x");
}
// contiguous and aligned for the kernels' 4-component loads
inline Tensor rows4(const Tensor& t) {
    const Tensor c = t.contiguous();
    return reinterpret_cast<uintptr_t>(c.data_ptr()) & 15 ? c.clone(at::MemoryFormat::Contiguous)
                                                          : c;
}
inline Tensor bytes_on(const Tensor& as, size_t n) {
    return torch::empty({(int64_t)((n + 15) / 16 * 16)},
                        torch::TensorOptions().dtype(torch::kUInt8).device(as.device()));
}

inline const Tensor* ptr_of(const OptTensor& t) { return t ? &*t : nullptr; }
// The kernels form no forward-mode derivatives: a tangent would be lost without a word, since a dual
// tensor need not require a gradient.
inline void refuse_tangent(const Tensor* t, const char* what) {
    TORCH_CHECK_NOT_IMPLEMENTED(!t || !t->defined() || !t->_fw_grad(/*level=*/0).defined(), what,
                                " has no forward-mode derivative");
}
inline void refuse_tangents(std::initializer_list<const Tensor*> all, const char* what) {
    if (!c10::AutogradState::get_tls_state().get_fw_grad_mode()) return;
    for (const Tensor* t : all) refuse_tangent(t, what);
}

inline void* opt_ptr(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
inline float* opt_f32(const Tensor& t) { return t.defined() ? t.data_ptr<float>() : nullptr; }

inline bool wants_grad(std::initializer_list<const Tensor*> all) {
    if (!at::GradMode::is_enabled()) return false;
    for (const Tensor* t : all)
        if (t && t->defined() && t->requires_grad()) return true;
    return false;
}
inline OptTensor opt_of(const Tensor& t) { return t.defined() ? OptTensor(t) : OptTensor(); }
inline Tensor tensor_of(const OptTensor& t) { return t ? *t : Tensor(); }

// The gradients as the graph takes them: under create_graph an error waits for whoever
// differentiates them again.
inline variable_list first_order(variable_list grads, bool create_graph, const char* what) {
    if (!create_graph) return grads;
    for (Tensor& g : grads)
        if (g.defined()) g = g.detach().set_requires_grad(true);
    const auto node = std::make_shared<torch::autograd::DelayedError>(
        std::string(what) + " is once_differentiable: its gradients have no gradients",
        (int64_t)grads.size());
    return node->apply(std::move(grads));
}

}  // namespace bmops
