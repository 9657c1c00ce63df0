// torch_memory.hpp — whether a tensor's address is one of memory.
#pragma once

#include <torch/extension.h>
#include <c10/core/impl/LocalDispatchKeySet.h>

namespace {

// torch.func.functionalize wraps tensors, outputs that are allocated under it among them, in ones
// whose storage is empty: of a view's address only the offset is left, a number that looks like a pointer.
inline void check_memory(const torch::Tensor& t, const char* name) {
    TORCH_CHECK(!t.defined() || !t.key_set().has(c10::DispatchKey::Functionalize), name,
                " is a functional wrapper without memory of its own: this library's calls cannot be functionalized");
}
inline void check_launch() {
    const auto active = c10::impl::tls_local_dispatch_key_set().included_;
    TORCH_CHECK(!active.has(c10::DispatchKey::FuncTorchDynamicLayerFrontMode) && !active.has(c10::DispatchKey::Functionalize),
                "this library's calls cannot be transformed by torch.func");
}

}  // namespace
