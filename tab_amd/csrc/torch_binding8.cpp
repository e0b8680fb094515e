// PyTorch front end of the 8-bit layers and of the norms around a block: checks, outputs from the caching allocator, one C ABI call an
// operator, and the autograd functions of tab_amd/nn.py.
#include <limits>

#include "torch_common.h"

using namespace tab_torch;

namespace {

using torch::Tensor;
using OptionalTensor = c10::optional<Tensor>;

int dtype_code(torch::ScalarType t, const char *name)
{
    switch (t) {
    case torch::kFloat32: return TAB_F32;
    case torch::kBFloat16: return TAB_BF16;
    case torch::kFloat16: return TAB_F16;
    default: TORCH_CHECK(false, name, " must have dtype torch.float32, torch.bfloat16 or torch.float16, got ", dtype_name(t));
    }
}

torch::ScalarType format_type(int format)
{
    TORCH_CHECK(format == TAB_E4M3 || format == TAB_E5M2, "format must be 0 (E4M3) or 1 (E5M2), got ", format);
    return format == TAB_E4M3 ? torch::kFloat8_e4m3fn : torch::kFloat8_e5m2;
}

int format_of(const Tensor &q, const char *name)
{
    TORCH_CHECK(q.scalar_type() == torch::kFloat8_e4m3fn || q.scalar_type() == torch::kFloat8_e5m2, name,
                " must have dtype torch.float8_e4m3fn or torch.float8_e5m2, got ", dtype_name(q.scalar_type()));
    return q.scalar_type() == torch::kFloat8_e4m3fn ? TAB_E4M3 : TAB_E5M2;
}

constexpr auto kScaleType = torch::kFloat8_e8m0fnu;

void check_device(const Tensor &t, const Tensor &like, const char *name)
{
    TORCH_CHECK(t.device().is_cuda(), name, " must be a CUDA tensor");
    TORCH_CHECK(t.device() == like.device(), "all tensors must be on the same device: ", name, " is on ", t.device());
}

// A contiguous tensor of rows * columns elements, or rows of a wider one; returns the row stride.
int64_t row_stride(const Tensor &t, int64_t rows, int64_t columns, const Tensor &like, const char *name)
{
    check_device(t, like, name);
    TORCH_CHECK(t.numel() == rows * columns, name, " has ", t.numel(), " elements, expected ", rows, " * ", columns);
    if (t.is_contiguous()) return columns;
    TORCH_CHECK(t.dim() == 2 && t.size(0) == rows && (columns == 1 || t.stride(1) == 1) && (rows == 1 || t.stride(0) >= columns), name,
                " must be contiguous or a matrix whose rows are");
    return rows == 1 ? columns : t.stride(0);
}

void check_whole(const Tensor &t, int64_t count, torch::ScalarType type, const Tensor &like, const char *name)
{
    check_device(t, like, name);
    TORCH_CHECK(t.is_contiguous(), name, " must be contiguous");
    TORCH_CHECK(t.scalar_type() == type, name, " must have dtype ", dtype_name(type), ", got ", dtype_name(t.scalar_type()));
    TORCH_CHECK(t.numel() == count, name, " has ", t.numel(), " elements, expected ", count);
}

const float *weights(const OptionalTensor &w, int64_t D, const Tensor &like, const char *name)
{
    if (!w) return nullptr;
    check_whole(*w, D, torch::kFloat32, like, name);
    return w->data_ptr<float>();
}

int64_t padded(int64_t K) { return (K + 127) / 128 * 128; }

// Q and S of a rows x columns matrix
std::array<Tensor, 2> packed_empty(int64_t rows, int64_t columns, int block_rows, int format, const Tensor &like)
{
    return {device_empty({rows, padded(columns)}, format_type(format), like),
            device_empty({padded(columns) / 128, block_rows == 1 ? rows : padded(rows) / 128}, kScaleType, like)};
}

void *data(const Tensor &t) { return t.defined() ? t.data_ptr() : nullptr; }

// {Q, S} and / or {QT, ST}
std::vector<Tensor> quantize8(const Tensor &X, int M, int K, int block_rows, int format, bool rows, bool columns)
{
    const int dtype = dtype_code(X.scalar_type(), "X");
    TORCH_CHECK(M > 0 && K > 0, "M and K must be positive");
    TORCH_CHECK(block_rows == 1 || block_rows == 128, "block_rows must be 1 or 128, got ", block_rows);
    const int64_t ld = row_stride(X, M, K, X, "X");
    const c10::hip::OptionalHIPGuardMasqueradingAsCUDA guard(X.device());
    std::array<Tensor, 2> q, qt;
    if (rows) q = packed_empty(M, K, block_rows, format, X);
    if (columns) qt = packed_empty(K, M, block_rows, format, X);
    check_status(tab_quantize8(X.data_ptr(), dtype, M, K, (long)ld, block_rows, format, data(q[0]), data(q[1]), data(qt[0]), data(qt[1]), current_stream(X)));
    if (!columns) return {q[0], q[1]};
    if (!rows) return {qt[0], qt[1]};
    return {q[0], q[1], qt[0], qt[1]};
}

std::vector<Tensor> TAB_Quantize8(const Tensor &X, int M, int K, int block_rows, int format) { return quantize8(X, M, K, block_rows, format, true, false); }
std::vector<Tensor> TAB_Quantize8Transposed(const Tensor &X, int M, int K, int block_rows, int format) { return quantize8(X, M, K, block_rows, format, false, true); }
std::vector<Tensor> TAB_Quantize8Both(const Tensor &X, int M, int K, int block_rows, int format) { return quantize8(X, M, K, block_rows, format, true, true); }

// Checks a packed weight; returns the rows of its blocks.
int check_weight(const Tensor &QW, const Tensor &SW, int N, int K, const Tensor &like)
{
    check_whole(QW, N * padded(K), torch::kFloat8_e4m3fn, like, "QW");
    check_device(SW, like, "SW");
    const int64_t KB = padded(K) / 128;
    const int block_rows = SW.numel() == KB * N ? 1 : 128;
    check_whole(SW, block_rows == 1 ? KB * N : KB * (padded(N) / 128), kScaleType, like, "SW");
    return block_rows;
}

void check_sizes(int M, int N, int K) { TORCH_CHECK(M > 0 && N > 0 && K > 0, "M, N, K must be positive"); }

template <typename CALL> void with_workspace(size_t bytes, const Tensor &like, CALL call)
{
    const hipStream_t stream = current_stream(like);
    if (bytes) call(Workspace(bytes, stream).get(), stream);
    else call(nullptr, stream);
}

Tensor TAB_Linear8(const Tensor &X, const Tensor &QW, const Tensor &SW, int M, int N, int K)
{
    const int dtype = dtype_code(X.scalar_type(), "X");
    check_sizes(M, N, K);
    const int64_t ld = row_stride(X, M, K, X, "X");
    const int block_rows = check_weight(QW, SW, N, K, X);
    const c10::hip::OptionalHIPGuardMasqueradingAsCUDA guard(X.device());
    auto Y = device_empty({M, N}, X.scalar_type(), X);
    const size_t bytes = tab_linear8_workspace_bytes(dtype, M, N, K);
    with_workspace(bytes, X, [&](void *ws, hipStream_t stream) {
        check_status(tab_linear8(X.data_ptr(), dtype, (long)ld, QW.data_ptr(), SW.data_ptr(), block_rows, M, N, K, Y.data_ptr(), ws, bytes, stream));
    });
    return Y;
}

Tensor TAB_Linear8Packed(const Tensor &QX, const Tensor &SX, const Tensor &QW, const Tensor &SW, int M, int N, int K, torch::ScalarType out_type)
{
    const int dtype = dtype_code(out_type, "the output"), format = format_of(QX, "QX");
    check_sizes(M, N, K);
    check_whole(QX, M * padded(K), QX.scalar_type(), QX, "QX");
    check_whole(SX, M * (padded(K) / 128), kScaleType, QX, "SX");
    const int block_rows = check_weight(QW, SW, N, K, QX);
    const c10::hip::OptionalHIPGuardMasqueradingAsCUDA guard(QX.device());
    auto Y = device_empty({M, N}, out_type, QX);
    const size_t bytes = tab_linear8_packed_workspace_bytes(dtype, M, N, K);
    with_workspace(bytes, QX, [&](void *ws, hipStream_t stream) {
        check_status(tab_linear8_packed(QX.data_ptr(), format, SX.data_ptr(), QW.data_ptr(), SW.data_ptr(), block_rows, M, N, K, Y.data_ptr(), dtype, ws,
                                        bytes, stream));
    });
    return Y;
}

// pybind11 knows torch.dtype as an object only
torch::ScalarType scalar_type(const pybind11::object &dtype)
{
    TORCH_CHECK_TYPE(THPDtype_Check(dtype.ptr()), "out_dtype must be a torch.dtype");
    return reinterpret_cast<THPDtype *>(dtype.ptr())->scalar_type;
}

// ---- norms ------------------------------------------------------------------------------------------------------------

enum { NORM_NONE = 0, NORM_PLAIN = 1, NORM_8BIT = 2 };

struct Gate {
    const void *data = nullptr;
    int dtype = TAB_F32, rows = 0;
    Gate(const OptionalTensor &gate, int64_t M, int64_t D, const Tensor &like)
    {
        if (!gate) return;
        check_device(*gate, like, "gate");
        TORCH_CHECK(gate->is_contiguous(), "gate must be contiguous");
        TORCH_CHECK(gate->scalar_type() == torch::kFloat32 || gate->scalar_type() == like.scalar_type(), "gate must have dtype torch.float32 or that of X, got ",
                    dtype_name(gate->scalar_type()));
        TORCH_CHECK(gate->numel() > 0 && gate->numel() % D == 0 && M % (gate->numel() / D) == 0, "gate has ", gate->numel(),
                    " elements, expected rows of D = ", D, ", their number a divisor of M = ", M);
        data = gate->data_ptr();
        dtype = dtype_code(gate->scalar_type(), "gate");
        rows = (int)(gate->numel() / D);
    }
};

// {R (with a block), H | QH, SH (by output)}
std::vector<Tensor> norm_forward(const Tensor &X, const OptionalTensor &Y, const OptionalTensor &gate, const OptionalTensor &w_post, const OptionalTensor &w_pre,
                                 double alpha, double eps, int M, int D, int output)
{
    const int dtype = dtype_code(X.scalar_type(), "X");
    TORCH_CHECK(M > 0 && D > 0, "M and D must be positive");
    TORCH_CHECK(output >= (Y ? NORM_NONE : NORM_PLAIN) && output <= NORM_8BIT, "output must be ", Y ? "0 (none), " : "", "1 (plain) or 2 (8 bit), got ", output);
    const int64_t ldx = row_stride(X, M, D, X, "X"), ldy = Y ? row_stride(*Y, M, D, X, "Y") : 0;
    TORCH_CHECK(!Y || Y->scalar_type() == X.scalar_type(), "Y must have X's dtype, got ", dtype_name(Y ? Y->scalar_type() : X.scalar_type()));
    const Gate g(gate, M, D, X);
    const float *post = weights(w_post, D, X, "w_post"), *pre = weights(w_pre, D, X, "w_pre");
    const c10::hip::OptionalHIPGuardMasqueradingAsCUDA guard(X.device());
    std::vector<Tensor> out;
    void *r = nullptr, *h = nullptr, *s = nullptr;
    if (Y) {
        out.push_back(device_empty({M, D}, X.scalar_type(), X));
        r = out.back().data_ptr();
    }
    if (output == NORM_PLAIN) {
        out.push_back(device_empty({M, D}, X.scalar_type(), X));
        h = out.back().data_ptr();
    } else if (output == NORM_8BIT) {
        auto packed = packed_empty(M, D, 1, TAB_E4M3, X);
        h = packed[0].data_ptr();
        s = packed[1].data_ptr();
        out.push_back(packed[0]);
        out.push_back(packed[1]);
    }
    check_status(tab_norm_residual(X.data_ptr(), (long)ldx, Y ? Y->data_ptr() : nullptr, (long)ldy, g.data, g.dtype, g.rows, post, pre, (float)alpha, (float)eps,
                                   dtype, M, D, r, h, s, current_stream(X)));
    return out;
}

std::vector<Tensor> TAB_NormResidual(const Tensor &X, const Tensor &Y, const OptionalTensor &gate, const OptionalTensor &w_post, const OptionalTensor &w_pre,
                                     double alpha, double eps, int M, int D, int output)
{
    return norm_forward(X, Y, gate, w_post, w_pre, alpha, eps, M, D, output);
}

std::vector<Tensor> TAB_Norm(const Tensor &X, const OptionalTensor &w, double eps, int M, int D, int output)
{
    return norm_forward(X, c10::nullopt, c10::nullopt, c10::nullopt, w, 1.0, eps, M, D, output);
}

// [dX, dY, dgate, dw_post, dw_pre], None for operands that are not there
std::vector<OptionalTensor> norm_backward(const OptionalTensor &dR, const OptionalTensor &dH, const Tensor &R, const OptionalTensor &Y, const OptionalTensor &gate,
                                          const OptionalTensor &w_post, const OptionalTensor &w_pre, double alpha, double eps, int M, int D)
{
    const int dtype = dtype_code(R.scalar_type(), "R");
    const int64_t count = (int64_t)M * D;
    TORCH_CHECK(M > 0 && D > 0, "M and D must be positive");
    TORCH_CHECK(dR || dH, "dR or dH must be given");
    check_whole(R, count, R.scalar_type(), R, "R");
    if (dR) check_whole(*dR, count, R.scalar_type(), R, "dR");
    if (dH) check_whole(*dH, count, R.scalar_type(), R, "dH");
    if (Y) check_whole(*Y, count, R.scalar_type(), R, "Y");
    const Gate g(gate, M, D, R);
    const float *post = weights(w_post, D, R, "w_post"), *pre = weights(w_pre, D, R, "w_pre");
    const c10::hip::OptionalHIPGuardMasqueradingAsCUDA guard(R.device());
    std::vector<OptionalTensor> out(5);
    out[0] = device_empty({M, D}, R.scalar_type(), R);
    if (Y) out[1] = device_empty({M, D}, R.scalar_type(), R);
    if (gate) out[2] = device_empty(gate->sizes(), gate->scalar_type(), R);
    if (w_post) out[3] = device_empty(w_post->sizes(), torch::kFloat32, R);
    if (w_pre) out[4] = device_empty(w_pre->sizes(), torch::kFloat32, R);
    auto at = [](const OptionalTensor &t) -> void * { return t ? t->data_ptr() : nullptr; };
    const size_t bytes = tab_norm_residual_backward_workspace_bytes(M, D, g.rows);
    with_workspace(bytes, R, [&](void *ws, hipStream_t stream) {
        check_status(tab_norm_residual_backward(at(dR), at(dH), R.data_ptr(), at(Y), g.data, g.dtype, g.rows, post, pre, (float)alpha, (float)eps, dtype, M, D,
                                                at(out[0]), at(out[1]), at(out[2]), static_cast<float *>(at(out[3])), static_cast<float *>(at(out[4])), ws, bytes,
                                                stream));
    });
    return out;
}

std::vector<OptionalTensor> TAB_NormResidualBackward(const OptionalTensor &dR, const OptionalTensor &dH, const Tensor &R, const Tensor &Y, const OptionalTensor &gate,
                                                     const OptionalTensor &w_post, const OptionalTensor &w_pre, double alpha, double eps, int M, int D)
{
    return norm_backward(dR, dH, R, Y, gate, w_post, w_pre, alpha, eps, M, D);
}

std::vector<OptionalTensor> TAB_NormBackward(const Tensor &dH, const Tensor &X, const OptionalTensor &w, double eps, int M, int D)
{
    const auto out = norm_backward(c10::nullopt, dH, X, c10::nullopt, c10::nullopt, c10::nullopt, w, 1.0, eps, M, D);
    return {out[0], out[4]};
}

// ---- autograd ---------------------------------------------------------------------------------------------------------

int as_size(int64_t v, const char *name)
{
    TORCH_CHECK(v > 0 && v <= std::numeric_limits<int>::max(), name, " must be positive and below 2^31, got ", v);
    return (int)v;
}

// There are no formulas for tangents (torch.autograd.forward_ad, one level): an input that has one is an error, as the kernels would drop it.
void no_tangent(std::initializer_list<const Tensor *> tensors)
{
    if (!c10::AutogradState::get_tls_state().get_fw_grad_mode()) return;
    for (const Tensor *t : tensors)
        TORCH_CHECK(!t || !t->defined() || !t->_fw_grad(0).defined(), "the 8-bit layers and the norms have no derivatives in forward mode (an input has a tangent)");
}

// The kernels' gradients are no graph: asking for their derivatives is an error, not a zero.
void no_second_derivative(const torch::autograd::variable_list &grads)
{
    TORCH_CHECK(!at::GradMode::is_enabled(), "the 8-bit layers and the norms have no second derivatives (create_graph)");
    for (const Tensor &g : grads) no_tangent({&g});
}

// Rows of the last dimension as a matrix with contiguous rows, and the same for the gradients.
Tensor matrix(const Tensor &x)
{
    const Tensor m = x.dim() == 2 ? x : x.reshape({-1, x.size(-1)});
    const bool rows = m.stride(1) == 1 && (m.size(0) == 1 || m.stride(0) >= m.size(1));
    return rows || m.size(1) == 1 ? (m.size(1) == 1 ? m.contiguous() : m) : m.contiguous();
}

// An output in its final shape that is no view: one of an autograd function that is a view may not be changed in place (a bias added, an activation).
Tensor shaped(const Tensor &t, c10::IntArrayRef sizes) { return t.sizes() == sizes ? t : at::_unsafe_view(t, sizes); }

// y = Q(x) Q(w)^T with gradients dx = Q(dy) Q(w), dw = Q(dy^T) Q(x^T)^T: three products of packed operands.  What the backward pass multiplies is
// packed in the forward pass, from the same reading of x and w.
struct Linear8Function : torch::autograd::Function<Linear8Function> {
    static Tensor forward(torch::autograd::AutogradContext *ctx, const Tensor &x, const Tensor &w, int64_t grad_format)
    {
        const bool need_dx = x.requires_grad(), need_dw = w.requires_grad();
        const Tensor x2 = matrix(x), w2 = matrix(w);
        const int M = as_size(x2.size(0), "rows of x"), K = as_size(x2.size(1), "columns of x"), N = as_size(w2.size(0), "rows of w");
        const auto qx = quantize8(x2, M, K, 1, TAB_E4M3, true, need_dw);
        const auto qw = quantize8(w2, N, K, 128, TAB_E4M3, true, need_dx);
        Tensor y = TAB_Linear8Packed(qx[0], qx[1], qw[0], qw[1], M, N, K, x.scalar_type());
        ctx->save_for_backward({need_dw ? qx[2] : Tensor(), need_dw ? qx[3] : Tensor(), need_dx ? qw[2] : Tensor(), need_dx ? qw[3] : Tensor()});
        ctx->saved_data["sizes"] = std::vector<int64_t>{M, N, K, grad_format, (int64_t)x.scalar_type(), (int64_t)w.scalar_type()};
        ctx->saved_data["shape"] = x.sizes().vec();
        auto shape = x.sizes().vec();
        shape.back() = N;
        return shaped(y, shape);
    }
    static torch::autograd::variable_list backward(torch::autograd::AutogradContext *ctx, const torch::autograd::variable_list &grads)
    {
        no_second_derivative(grads);
        const auto saved = ctx->get_saved_variables();
        const auto sizes = ctx->saved_data["sizes"].toIntVector();
        const int M = (int)sizes[0], N = (int)sizes[1], K = (int)sizes[2], format = (int)sizes[3];
        const bool need_dw = saved[0].defined(), need_dx = saved[2].defined();
        const Tensor dy = matrix(grads[0]);
        const auto q = quantize8(dy, M, N, 1, format, need_dx, need_dw);
        Tensor dx, dw;
        if (need_dx) dx = TAB_Linear8Packed(q[0], q[1], saved[2], saved[3], M, K, N, (torch::ScalarType)sizes[4]).view(ctx->saved_data["shape"].toIntVector());
        if (need_dw) {
            const size_t at = need_dx ? 2 : 0;
            dw = TAB_Linear8Packed(q[at], q[at + 1], saved[0], saved[1], N, K, M, (torch::ScalarType)sizes[5]);
        }
        return {dx, dw, Tensor()};
    }
};

bool wants_gradient(std::initializer_list<const Tensor *> tensors)
{
    if (!at::GradMode::is_enabled()) return false;
    for (const Tensor *t : tensors)
        if (t && t->requires_grad()) return true;
    return false;
}

Tensor linear8(const Tensor &x, const Tensor &w, int grad_format)
{
    dtype_code(x.scalar_type(), "x");
    dtype_code(w.scalar_type(), "w");
    format_type(grad_format);
    TORCH_CHECK(x.dim() >= 1 && w.dim() == 2 && x.size(-1) == w.size(1), "x (..., K) and w (N, K) must agree in K, got ", x.sizes(), " and ", w.sizes());
    TORCH_CHECK(x.numel() > 0 && w.numel() > 0, "x and w must not be empty, got ", x.sizes(), " and ", w.sizes());
    no_tangent({&x, &w});
    check_device(w, x, "w");
    if (wants_gradient({&x, &w})) return Linear8Function::apply(x, w, (int64_t)grad_format);
    const Tensor x2 = matrix(x), w2 = matrix(w);
    const int M = as_size(x2.size(0), "rows of x"), K = as_size(x2.size(1), "columns of x"), N = as_size(w2.size(0), "rows of w");
    const auto qw = quantize8(w2, N, K, 128, TAB_E4M3, true, false);
    auto shape = x.sizes().vec();
    shape.back() = N;
    return TAB_Linear8(x2, qw[0], qw[1], M, N, K).view(shape);
}

// nn.Linear8.forward
Tensor linear8_packed_weight(const Tensor &x, const Tensor &QW, const Tensor &SW, int N, int K)
{
    TORCH_CHECK(x.dim() >= 1 && x.size(-1) == K && x.numel() > 0, "input must be (..., ", K, ") and not empty, got ", x.sizes());
    no_tangent({&x});
    TORCH_CHECK(!wants_gradient({&x}), "a packed weight is for inference: take nn.linear8 for training");
    const Tensor x2 = matrix(x);
    auto shape = x.sizes().vec();
    shape.back() = N;
    return TAB_Linear8(x2, QW, SW, as_size(x2.size(0), "rows of the input"), N, K).view(shape);
}

OptionalTensor optional(const Tensor &t) { return t.defined() ? OptionalTensor(t) : c10::nullopt; }
Tensor defined(const OptionalTensor &t) { return t ? *t : Tensor(); }

struct NormFunction : torch::autograd::Function<NormFunction> {
    // Returns {R, H}, {R} or {H}
    static torch::autograd::variable_list forward(torch::autograd::AutogradContext *ctx, const Tensor &x, const OptionalTensor &y, const OptionalTensor &gate,
                                                  const OptionalTensor &w_post, const OptionalTensor &w_pre, double alpha, double eps, int64_t output)
    {
        const Tensor x2 = matrix(x);
        const OptionalTensor y2 = y ? OptionalTensor(matrix(*y)) : y;
        const int M = as_size(x2.size(0), "rows of x"), D = as_size(x2.size(1), "columns of x");
        auto out = norm_forward(x2, y2, gate, w_post, w_pre, alpha, eps, M, D, (int)output);
        for (Tensor &t : out) t = shaped(t, x.sizes());
        ctx->save_for_backward({y ? out[0] : x2.contiguous(), y ? y2->contiguous() : Tensor(), defined(gate), defined(w_post), defined(w_pre)});
        ctx->saved_data["alpha"] = alpha;
        ctx->saved_data["eps"] = eps;
        ctx->saved_data["output"] = output;
        ctx->set_materialize_grads(false);
        return out;
    }
    static torch::autograd::variable_list backward(torch::autograd::AutogradContext *ctx, const torch::autograd::variable_list &grads)
    {
        no_second_derivative(grads);
        const auto saved = ctx->get_saved_variables();
        const bool block = saved[1].defined();
        const int64_t output = ctx->saved_data["output"].toInt();
        const Tensor none, dr = block ? grads[0] : none, dh = output == NORM_NONE ? none : grads[block ? 1 : 0];
        if (!dr.defined() && !dh.defined()) return {none, none, none, none, none, none, none, none};
        const Tensor &like = dr.defined() ? dr : dh;
        const int D = (int)like.size(-1), M = (int)(like.numel() / D);
        auto whole = [](const Tensor &t) { return t.defined() ? OptionalTensor(t.contiguous()) : c10::nullopt; };
        const auto out = norm_backward(whole(dr), whole(dh), saved[0], optional(saved[1]), optional(saved[2]), optional(saved[3]), optional(saved[4]),
                                       ctx->saved_data["alpha"].toDouble(), ctx->saved_data["eps"].toDouble(), M, D);
        auto like_it = [&](const OptionalTensor &t) { return t ? t->view(like.sizes()) : Tensor(); };
        return {like_it(out[0]), like_it(out[1]), defined(out[2]), defined(out[3]), defined(out[4]), none, none, none};
    }
};

// Weights and gates as the kernels take them: contiguous (a gate is often a part of a wider modulation), weights of a module that was converted to 16 bits
// as fp32, and gates of 16 bits that are not x's.  All of it is differentiable.
OptionalTensor taken(const OptionalTensor &w, torch::ScalarType kept = torch::kFloat32)
{
    if (!w) return w;
    const auto type = w->scalar_type();
    const bool widen = type != kept && (type == torch::kBFloat16 || type == torch::kFloat16);
    return (widen ? w->to(torch::kFloat32) : *w).contiguous();
}

// A row of the kernels' gate holds for consecutive rows of x.  Torch would broadcast a gate of (1, S, D) over the first dimension of x: refused.
void check_gate(const Tensor &gate, c10::IntArrayRef x)
{
    const int64_t dims = (int64_t)x.size();
    if (gate.dim() != dims || dims < 3) return;
    int64_t d = 0;
    while (d < dims - 1 && gate.size(d) == x[d]) d++;
    for (; d < dims - 1; d++)
        TORCH_CHECK(gate.size(d) == 1, "a row of the gate holds for consecutive rows of x: sizes other than 1 must be x's first ones, got ", gate.sizes(), " and ", x);
}

// nn.norm_residual: x (..., D) and y of its shape
std::vector<Tensor> norm_residual(const Tensor &x, const OptionalTensor &y, const OptionalTensor &any_gate, const OptionalTensor &any_post, const OptionalTensor &any_pre,
                                  double alpha, double eps, int output)
{
    TORCH_CHECK(x.dim() >= 1 && x.numel() > 0, "x must not be empty, got ", x.sizes());
    TORCH_CHECK(!y || y->sizes() == x.sizes(), "y must have x's shape, got ", y ? y->sizes() : x.sizes(), " and ", x.sizes());
    TORCH_CHECK(y || output != NORM_NONE, "without a block there is nothing to do but the norm");
    if (any_gate) check_gate(*any_gate, x.sizes());
    const auto at = [](const OptionalTensor &t) { return t ? &*t : nullptr; };
    no_tangent({&x, at(y), at(any_gate), at(any_post), at(any_pre)});
    const OptionalTensor gate = taken(any_gate, x.scalar_type()), w_post = taken(any_post), w_pre = taken(any_pre);
    if (output != NORM_8BIT && wants_gradient({&x, at(y), at(gate), at(w_post), at(w_pre)}))
        return NormFunction::apply(x, y, gate, w_post, w_pre, alpha, eps, (int64_t)output);
    TORCH_CHECK(!wants_gradient({&x, at(y), at(gate), at(w_post), at(w_pre)}), "the packed output has no gradient: take the plain one and linear8 for training");
    const Tensor x2 = matrix(x);
    auto out = norm_forward(x2, y ? OptionalTensor(matrix(*y)) : y, gate, w_post, w_pre, alpha, eps, as_size(x2.size(0), "rows of x"),
                            as_size(x2.size(1), "columns of x"), output);
    for (size_t i = 0; i < out.size() - (output == NORM_8BIT ? 2 : 0); i++) out[i] = out[i].view(x.sizes());
    return out;
}

}  // namespace

void bind_layers8(pybind11::module_ &m)
{
    using pybind11::arg;
    m.def("Quantize8", &TAB_Quantize8, "X packed in 8 bits with a power-of-two scale per block of 128: [Q, S]", arg("X"), arg("M"), arg("K"), arg("block_rows") = 1,
          arg("format") = (int)TAB_E4M3);
    m.def("Quantize8Transposed", &TAB_Quantize8Transposed, "X transposed, packed: [QT, ST]", arg("X"), arg("M"), arg("K"), arg("block_rows") = 1,
          arg("format") = (int)TAB_E4M3);
    m.def("Quantize8Both", &TAB_Quantize8Both, "Both from one reading of X: [Q, S, QT, ST]", arg("X"), arg("M"), arg("K"), arg("block_rows") = 1,
          arg("format") = (int)TAB_E4M3);
    m.def("Linear8", &TAB_Linear8, "X, quantized on the way, times packed weights", arg("X"), arg("QW"), arg("SW"), arg("M"), arg("N"), arg("K"));
    m.def(
        "Linear8Packed",
        [](const Tensor &QX, const Tensor &SX, const Tensor &QW, const Tensor &SW, int M, int N, int K, const pybind11::object &out_dtype) {
            return TAB_Linear8Packed(QX, SX, QW, SW, M, N, K, scalar_type(out_dtype));
        },
        "Product of two packed operands");
    m.def("Norm", &TAB_Norm, "rms norm of the rows of X, plain or packed");
    m.def("NormResidual", &TAB_NormResidual, "norm after a block, gate, scaled residual and the norm before the next block");
    m.def("NormResidualBackward", &TAB_NormResidualBackward, "gradients of NormResidual");
    m.def("NormBackward", &TAB_NormBackward, "gradients of Norm");
    m.def("linear8", &linear8, "nn.linear8");
    m.def("linear8_packed_weight", &linear8_packed_weight, "nn.Linear8.forward");
    m.def("check_gate", [](const Tensor &gate, const std::vector<int64_t> &x) { check_gate(gate, x); }, "whether a gate of x's dimensions holds for consecutive rows");
    m.def("norm_residual", &norm_residual, "nn.norm_residual");
}
