// torch_checks.hpp — what the torch surfaces of the operators share: status and argument
// checks, the current stream.
#pragma once

#include <torch/extension.h>
#include <c10/core/AutogradState.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/jit/frontend/tracer.h>

#include "../../include/ra_spmm.h"
#include "torch_memory.hpp"

namespace {

using torch::Tensor;
using OptTensor = c10::optional<Tensor>;

inline ra_stream_t current_stream() {
    check_launch();
    return reinterpret_cast<ra_stream_t>(c10::hip::getCurrentHIPStream().stream());
}

inline void check(ra_status s, const char* what) {
    TORCH_CHECK(s == RA_OK, what, " failed: ", ra_status_string(s), ": ", ra_last_error());
}

inline int dtype_of(const Tensor& t, const char* name) {
    if (t.scalar_type() == torch::kFloat32) return RA_DTYPE_F32;
    if (t.scalar_type() == torch::kFloat16) return RA_DTYPE_F16;
    if (t.scalar_type() == torch::kBFloat16) return RA_DTYPE_BF16;
    TORCH_CHECK(false, name, " must be float32, float16 or bfloat16");
    return -1;
}

// A tensor with a tangent need not require a gradient: without this check the result would be
// one whose tangent is missing.
struct Named {
    const Tensor& t;
    const char* name;
};
inline void check_no_tangents(std::initializer_list<Named> of) {
    if (!c10::AutogradState::get_tls_state().get_fw_grad_mode()) return;
    for (const Named& n : of)
        TORCH_CHECK(!n.t.defined() || !n.t._fw_grad(0).defined(), n.name,
                    " carries a forward-mode tangent, this operator has reverse-mode derivatives only");
}

// Tracers record torch's own operations: of a call here they would keep the outputs' allocation
// and no launch, and a replay would return memory that nobody wrote.
inline void check_no_tracer(const char* what) {
    TORCH_CHECK(!torch::jit::tracer::isTracing(), what, " cannot be traced: torch.jit.trace does not see its launches");
}
inline void check_no_proxies(const char* name) {
    using c10::impl::TorchDispatchModeKey;
    using c10::impl::TorchDispatchModeTLS;
    if (!TorchDispatchModeTLS::any_modes_set()) return;
    TORCH_CHECK(!TorchDispatchModeTLS::get_mode(TorchDispatchModeKey::PROXY) && !TorchDispatchModeTLS::get_mode(TorchDispatchModeKey::FAKE),
                name, ": this operator cannot be traced (make_fx, torch.export or fake tensors)");
}

inline void check_values(const Tensor& t, const char* name) {
    check_no_tangents({{t, name}});
    check_memory(t, name);
    TORCH_CHECK(t.is_cuda(), name, " must be a CUDA tensor");
    TORCH_CHECK(!t.is_neg(), name, " is a view of the negated values (resolve_neg() gives them)");
}

// A call's first tensor, and the others.
inline void check_cuda(const Tensor& t, const char* name) {
    check_no_proxies(name);
    check_values(t, name);
}
inline void check_on(const Tensor& t, const char* name, const torch::Device& dev) {
    check_values(t, name);
    TORCH_CHECK(t.device() == dev, name, " must be on ", dev, ", is on ", t.device());
}

inline const float* f32_vector(const Tensor& t, const char* name, int64_t n, const torch::Device& dev) {
    check_on(t, name, dev);
    TORCH_CHECK(t.scalar_type() == torch::kFloat32, name, " must be float32");
    TORCH_CHECK(t.dim() == 1 && t.numel() == n, name, " must have shape [", n, "], has ", t.sizes());
    TORCH_CHECK(t.is_contiguous(), name, " must be contiguous");
    return t.data_ptr<float>();
}

// Distance between the rows of t, whose other dimensions have to be contiguous.
inline int64_t row_stride(const Tensor& t, const char* name) {
    int64_t run = 1;
    for (int64_t d = t.dim() - 1; d > 0; --d) {
        TORCH_CHECK(t.size(d) <= 1 || t.stride(d) == run, name, " must be contiguous within its rows");
        run *= t.size(d);
    }
    if (t.size(0) <= 1) return run;
    TORCH_CHECK(t.stride(0) >= run, name, " must not have rows that overlap");
    return t.stride(0);
}

}  // namespace
