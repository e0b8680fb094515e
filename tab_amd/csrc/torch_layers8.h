// What the bindings of the 8-bit and 4-bit layers, the norms and the experts share: types, checks of tensors, packed operands, workspaces.
#pragma once
#include <limits>

#include "torch_common.h"

namespace tab_torch {

using torch::Tensor;
using OptionalTensor = c10::optional<Tensor>;

inline int dtype_code(torch::ScalarType t, const char *name)
{
    switch (t) {
    case torch::kFloat32: return TAB_F32;
    case torch::kBFloat16: return TAB_BF16;
    case torch::kFloat16: return TAB_F16;
    default: TORCH_CHECK(false, name, " must have dtype torch.float32, torch.bfloat16 or torch.float16, got ", dtype_name(t));
    }
}

inline torch::ScalarType format_type(int format)
{
    TORCH_CHECK(format == TAB_E4M3 || format == TAB_E5M2, "format must be 0 (E4M3) or 1 (E5M2), got ", format);
    return format == TAB_E4M3 ? torch::kFloat8_e4m3fn : torch::kFloat8_e5m2;
}

inline int format_of(const Tensor &q, const char *name)
{
    TORCH_CHECK(q.scalar_type() == torch::kFloat8_e4m3fn || q.scalar_type() == torch::kFloat8_e5m2, name,
                " must have dtype torch.float8_e4m3fn or torch.float8_e5m2, got ", dtype_name(q.scalar_type()));
    return q.scalar_type() == torch::kFloat8_e4m3fn ? TAB_E4M3 : TAB_E5M2;
}

constexpr auto kScaleType = torch::kFloat8_e8m0fnu;

inline void check_device(const Tensor &t, const Tensor &like, const char *name)
{
    TORCH_CHECK(t.device().is_cuda(), name, " must be a CUDA tensor");
    TORCH_CHECK(t.device() == like.device(), "all tensors must be on the same device: ", name, " is on ", t.device());
}

// A contiguous tensor of rows * columns elements, or rows of a wider one; returns the row stride.
inline int64_t row_stride(const Tensor &t, int64_t rows, int64_t columns, const Tensor &like, const char *name)
{
    check_device(t, like, name);
    TORCH_CHECK(t.numel() == rows * columns, name, " has ", t.numel(), " elements, expected ", rows, " * ", columns);
    if (t.is_contiguous()) return columns;
    TORCH_CHECK(t.dim() == 2 && t.size(0) == rows && (columns == 1 || t.stride(1) == 1) && (rows == 1 || t.stride(0) >= columns), name,
                " must be contiguous or a matrix whose rows are");
    return rows == 1 ? columns : t.stride(0);
}

inline void check_whole(const Tensor &t, int64_t count, torch::ScalarType type, const Tensor &like, const char *name)
{
    check_device(t, like, name);
    TORCH_CHECK(t.is_contiguous(), name, " must be contiguous");
    TORCH_CHECK(t.scalar_type() == type, name, " must have dtype ", dtype_name(type), ", got ", dtype_name(t.scalar_type()));
    TORCH_CHECK(t.numel() == count, name, " has ", t.numel(), " elements, expected ", count);
}

inline int64_t padded(int64_t K) { return (K + 127) / 128 * 128; }

// Q and S of a rows x columns matrix
inline std::array<Tensor, 2> packed_empty(int64_t rows, int64_t columns, int block_rows, int format, const Tensor &like)
{
    return {device_empty({rows, padded(columns)}, format_type(format), like),
            device_empty({padded(columns) / 128, block_rows == 1 ? rows : padded(rows) / 128}, kScaleType, like)};
}

inline void *data(const Tensor &t) { return t.defined() ? t.data_ptr() : nullptr; }

inline void check_sizes(int M, int N, int K) { TORCH_CHECK(M > 0 && N > 0 && K > 0, "M, N, K must be positive"); }

template <typename CALL> void with_workspace(size_t bytes, const Tensor &like, CALL call)
{
    const hipStream_t stream = current_stream(like);
    if (bytes) call(Workspace(bytes, stream).get(), stream);
    else call(nullptr, stream);
}

// pybind11 knows torch.dtype as an object only
inline torch::ScalarType scalar_type(const pybind11::object &dtype)
{
    TORCH_CHECK_TYPE(THPDtype_Check(dtype.ptr()), "out_dtype must be a torch.dtype");
    return reinterpret_cast<THPDtype *>(dtype.ptr())->scalar_type;
}

inline int as_size(int64_t v, const char *name)
{
    TORCH_CHECK(v > 0 && v <= std::numeric_limits<int>::max(), name, " must be positive and below 2^31, got ", v);
    return (int)v;
}

// Rows of the last dimension as a matrix with contiguous rows, and the same for the gradients.
inline Tensor matrix(const Tensor &x)
{
    const Tensor m = x.dim() == 2 ? x : x.reshape({-1, x.size(-1)});
    const bool rows = m.stride(1) == 1 && (m.size(0) == 1 || m.stride(0) >= m.size(1));
    return rows || m.size(1) == 1 ? (m.size(1) == 1 ? m.contiguous() : m) : m.contiguous();
}

// An output in its final shape that is no view: one of an autograd function that is a view may not be changed in place (a bias added, an activation).
inline Tensor shaped(const Tensor &t, c10::IntArrayRef sizes) { return t.sizes() == sizes ? t : at::_unsafe_view(t, sizes); }

inline bool wants_gradient(std::initializer_list<const Tensor *> tensors)
{
    if (!at::GradMode::is_enabled()) return false;
    for (const Tensor *t : tensors)
        if (t && t->requires_grad()) return true;
    return false;
}

// There are no formulas for tangents (torch.autograd.forward_ad, one level): an input that has one is an error, as the kernels would drop it.
inline void no_tangent(std::initializer_list<const Tensor *> tensors)
{
    if (!c10::AutogradState::get_tls_state().get_fw_grad_mode()) return;
    for (const Tensor *t : tensors)
        TORCH_CHECK(!t || !t->defined() || !t->_fw_grad(0).defined(), "this layer has no derivatives in forward mode (an input has a tangent)");
}

// The kernels' gradients are no graph: asking for their derivatives is an error, not a zero.
inline void no_second_derivative(const torch::autograd::variable_list &grads)
{
    TORCH_CHECK(!at::GradMode::is_enabled(), "this layer has no second derivatives (create_graph)");
    for (const Tensor &g : grads) no_tangent({&g});
}

}  // namespace tab_torch
