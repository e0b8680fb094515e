// What the sources of the PyTorch extension share: the checks of the reference's boundary (TAB_GPU.cpp:7-9), errors of the C ABI, the
// current stream, outputs and scratch from the caching allocator.
#pragma once
#include <torch/extension.h>

#include <ATen/hip/EmptyTensor.h>
#include <ATen/hip/impl/HIPGuardImplMasqueradingAsCUDA.h>
#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>
#include <c10/hip/HIPCachingAllocator.h>

#include <array>
#include <memory>
#include <stdexcept>
#include <tuple>
#include <vector>

#include "../../include/tab_amd.h"

// CHECK_INPUT of the reference (TAB_GPU.cpp:7-9)
#define CHECK_CUDA(x) TORCH_CHECK(x.device().is_cuda(), #x " must be a CUDA tensor")
#define CHECK_CONTIGUOUS(x) TORCH_CHECK(x.is_contiguous(), #x " must be contiguous")
#define CHECK_INPUT(x) \
    CHECK_CUDA(x);     \
    CHECK_CONTIGUOUS(x)
// The reference converts dtypes with .toType() on a temporary (TAB_GEMM.cu:279-280,341-347),
// which dangles whenever a conversion really happens; exact dtypes are required instead.
#define CHECK_DTYPE(x, t) \
    TORCH_CHECK(x.scalar_type() == torch::t, #x " must have dtype ", dtype_name(torch::t), ", got ", dtype_name(x.scalar_type()))

namespace tab_torch {

inline std::string dtype_name(torch::ScalarType t)
{
    switch (t) {
    case torch::kFloat32: return "torch.float32";
    case torch::kInt64: return "torch.int64";
    case torch::kInt32: return "torch.int32";
    default: return std::string("torch.") + c10::toString(t);
    }
}

// A negative status of a C ABI call; Python sees tab_amd.TabError (a RuntimeError).
struct StatusError : std::runtime_error {
    using std::runtime_error::runtime_error;
};

inline void check_status(int status)
{
    if (status != TAB_OK) throw StatusError(std::string(tab_status_string(status)) + ": " + tab_last_error());
}

inline hipStream_t current_stream(const torch::Tensor &t)
{
    return c10::hip::getCurrentHIPStreamMasqueradingAsCUDA(t.device().index()).stream();
}

// Uninitialised device tensor, straight from the caching allocator: torch::empty's way through the dispatcher costs
// 0.73 us a tensor, this 0.47, beside 2.3 us for a kernel launch.
inline torch::Tensor device_empty(c10::IntArrayRef sizes, torch::ScalarType dtype, const torch::Tensor &like)
{
    return at::detail::empty_cuda(sizes, dtype, like.device(), c10::nullopt);
}

// Device scratch of one call (0.2 us, no tensor around it).  Given back when the call returns: the allocator hands the
// block only to later work of the same stream.
class Workspace {
public:
    Workspace(size_t bytes, hipStream_t stream)
        : ptr_(c10::hip::HIPCachingAllocator::raw_alloc_with_stream(bytes, stream)) {}
    ~Workspace() { c10::hip::HIPCachingAllocator::raw_delete(ptr_); }
    Workspace(const Workspace &) = delete;
    Workspace &operator=(const Workspace &) = delete;
    void *get() const { return ptr_; }

private:
    void *ptr_;
};

}  // namespace tab_torch
