// What the PyTorch front end's operators share: descriptors of tensors, the
// current stream, errors, and the refusals of what autograd could not follow.
#pragma once
#include <torch/extension.h>
#include <ATen/cuda/CUDAGeneratorImpl.h>
#include <torch/csrc/autograd/function.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/saved_variable.h>
#include <torch/csrc/jit/frontend/tracer.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>

#include <algorithm>
#include <memory>
#include <mutex>
#include <stdexcept>
#include <string>
#include <vector>

#include "groupconv.h"

namespace front_end {

inline gc_tensor describe(const at::Tensor &t) {
    gc_tensor d{};
    d.data = t.data_ptr();
    d.bytes = static_cast<uint64_t>(t.numel()) * t.element_size();
    d.dtype = t.scalar_type() == at::kFloat ? GC_F32 : t.scalar_type() == at::kDouble ? GC_F64 : -1;
    d.device = t.is_cuda() ? GC_CUDA : t.is_cpu() ? GC_CPU : -1;
    d.device_index = t.is_cuda() ? t.get_device() : 0;
    d.rank = static_cast<int32_t>(t.dim());
    for (int i = 0; i < 4 && i < t.dim(); ++i) {
        d.dims[i] = t.size(i);
        d.strides[i] = t.stride(i);
    }
    return d;
}

// A tracer records what passes through the dispatcher: of these calls only the
// output's allocation, so that the recorded graph would return memory that
// nothing writes.
inline void no_tracing() {
    if (torch::jit::tracer::isTracing() ||
        c10::impl::TorchDispatchModeTLS::get_mode(c10::impl::TorchDispatchModeKey::PROXY).has_value())
        throw std::runtime_error("this operation cannot be traced");
}

[[noreturn]] inline void fail(int status) {
    throw std::runtime_error("gc_status " + std::to_string(status) + ": " + gc_last_error());
}

// As describe(), for the entry points that also take 16-bit types and strided
// views: bytes covers the view from its first to its last element.
inline gc_tensor describe_view(const at::Tensor &t) {
    gc_tensor d = describe(t);
    if (t.scalar_type() == at::kHalf) d.dtype = GC_B200_F16;
    if (t.scalar_type() == at::kBFloat16) d.dtype = GC_B200_BF16;
    if (t.numel() > 0) {
        int64_t last = 1;
        for (int64_t i = 0; i < t.dim(); ++i) last += (t.size(i) - 1) * t.stride(i);
        d.bytes = static_cast<uint64_t>(last) * t.element_size();
    }
    return d;
}

inline void *stream_of(const at::Tensor &t) {
    return t.is_cuda() ? static_cast<void *>(c10::cuda::getCurrentCUDAStream(t.get_device()).stream()) : nullptr;
}

inline at::Tensor workspace_of(uint64_t bytes, const at::Tensor &like) {
    return bytes == 0 ? at::Tensor()
                      : at::empty({static_cast<int64_t>(bytes)}, like.options().dtype(at::kByte).memory_format(
                                                                     at::MemoryFormat::Contiguous));
}

inline void no_double_backward() {
    if (at::GradMode::is_enabled())
        throw std::runtime_error("the gradient of this operation is not differentiable (create_graph)");
}

// Asked of every operand whether it requires a gradient or not: the primal of a
// dual tensor usually does not, and its tangent would be lost.
inline void no_forward_mode(const at::Tensor &t) {
    if (t.defined() && t._fw_grad(/*level=*/0).defined())
        throw std::runtime_error("this operation has no forward-mode derivative");
}

inline bool wants_grad(const at::Tensor &t) { return t.defined() && t.requires_grad(); }

}  // namespace front_end
