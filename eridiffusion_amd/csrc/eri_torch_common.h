/* What the native modules of the Python face share: making tensors past the dispatcher. */
#pragma once
#include <ATen/ATen.h>
#include <ATen/EmptyTensor.h>
#include <ATen/detail/CUDAHooksInterface.h>
#include <c10/core/impl/LocalDispatchKeySet.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>

namespace eri_face {

/* Whether nothing wants to see or to change the tensors that are made now: no dispatch mode, transform or tracer, no
 * filling of uninitialised memory. */
inline bool factories_are_plain() {
    if (c10::impl::TorchDispatchModeTLS::any_modes_set()) return false;
    if (c10::impl::tls_local_dispatch_key_set().included_ != c10::default_included_set) return false;
    return !(at::globalContext().deterministicAlgorithms() && at::globalContext().deterministicFillUninitializedMemory());
}

/* Tensors like others, on their devices: what at::empty_strided makes on a device, past the dispatcher. */
struct Outputs {
    const bool direct = factories_are_plain();
    c10::Allocator *const allocator = direct ? at::detail::getCUDAHooks().getCUDADeviceAllocator() : nullptr;
    c10::OptionalDeviceGuard guard;
    at::Tensor like(const at::Tensor &t) {
        if (!direct) return at::empty_strided(t.sizes(), t.strides(), t.options());
        if (guard.current_device() != t.device()) guard.reset_device(t.device());
        return at::detail::empty_strided_generic(t.sizes(), t.strides(), allocator, c10::DispatchKeySet(c10::DispatchKey::CUDA), t.scalar_type());
    }
    /* A new contiguous tensor on t's device. */
    at::Tensor empty(at::IntArrayRef sizes, at::ScalarType dtype, const at::Tensor &t) {
        if (!direct) return at::empty(sizes, t.options().dtype(dtype));
        if (guard.current_device() != t.device()) guard.reset_device(t.device());
        return at::detail::empty_generic(sizes, allocator, c10::DispatchKeySet(c10::DispatchKey::CUDA), dtype, std::nullopt);
    }
};

} // namespace eri_face
