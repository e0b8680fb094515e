// PyTorch front end of the 4-bit layers and of layers of experts: checks, outputs from the caching allocator, C ABI calls, and the autograd functions
// of tab_amd/nn.py.
#include "torch_layers8.h"

using namespace tab_torch;

namespace {

constexpr auto kFourBits = torch::kFloat4_e2m1fn_x2;  // two numbers an element

const int *int32s(const Tensor &t, int64_t count, const Tensor &like, const char *name)
{
    check_whole(t, count, torch::kInt32, like, name);
    return t.data_ptr<int>();
}
const int *int32s(const OptionalTensor &t, int64_t count, const Tensor &like, const char *name) { return t ? int32s(*t, count, like, name) : nullptr; }

// ---- 4-bit layers -----------------------------------------------------------------------------------------------------

std::vector<Tensor> quantize4(const Tensor &X, int E, int M, int K, bool batch)
{
    const int dtype = dtype_code(X.scalar_type(), "X");
    TORCH_CHECK(E > 0 && M > 0 && K > 0, batch ? "E, N and K must be positive" : "M and K must be positive");
    const int64_t ld = row_stride(X, (int64_t)E * M, K, X, "X"), KB = padded(K) / 128;
    const c10::hip::OptionalHIPGuardMasqueradingAsCUDA guard(X.device());
    auto Q = batch ? device_empty({E, M, padded(K) / 2}, kFourBits, X) : device_empty({M, padded(K) / 2}, kFourBits, X);
    auto S = batch ? device_empty({E, KB, M, 4}, kScaleType, X) : device_empty({KB, M, 4}, kScaleType, X);
    check_status(tab_quantize4(X.data_ptr(), dtype, E, M, K, (long)ld, Q.data_ptr(), S.data_ptr(), current_stream(X)));
    return {Q, S};
}

std::vector<Tensor> TAB_Quantize4(const Tensor &X, int M, int K) { return quantize4(X, 1, M, K, false); }

void check_weight4(const Tensor &QW, const Tensor &SW, int64_t E, int N, int K, const Tensor &like)
{
    check_whole(QW, E * N * (padded(K) / 2), kFourBits, like, "QW");
    check_whole(SW, E * N * (padded(K) / 32), kScaleType, like, "SW");
}

Tensor TAB_Linear4(const Tensor &X, const Tensor &QW, const Tensor &SW, int M, int N, int K)
{
    const int dtype = dtype_code(X.scalar_type(), "X");
    check_sizes(M, N, K);
    const int64_t ld = row_stride(X, M, K, X, "X");
    check_weight4(QW, SW, 1, N, K, X);
    const c10::hip::OptionalHIPGuardMasqueradingAsCUDA guard(X.device());
    auto Y = device_empty({M, N}, X.scalar_type(), X);
    const size_t bytes = tab_linear4_workspace_bytes(dtype, M, N, K);
    with_workspace(bytes, X, [&](void *ws, hipStream_t stream) {
        check_status(tab_linear4(X.data_ptr(), dtype, (long)ld, QW.data_ptr(), SW.data_ptr(), M, N, K, Y.data_ptr(), ws, bytes, stream));
    });
    return Y;
}

Tensor TAB_Linear4Packed(const Tensor &QX, const Tensor &SX, const Tensor &QW, const Tensor &SW, int M, int N, int K, torch::ScalarType out_type)
{
    const int dtype = dtype_code(out_type, "the output");
    check_sizes(M, N, K);
    check_whole(QX, M * padded(K), torch::kFloat8_e4m3fn, QX, "QX");
    check_whole(SX, M * (padded(K) / 128), kScaleType, QX, "SX");
    check_weight4(QW, SW, 1, N, K, QX);
    const c10::hip::OptionalHIPGuardMasqueradingAsCUDA guard(QX.device());
    auto Y = device_empty({M, N}, out_type, QX);
    const size_t bytes = tab_linear4_packed_workspace_bytes(dtype, M, N, K);
    with_workspace(bytes, QX, [&](void *ws, hipStream_t stream) {
        check_status(tab_linear4_packed(QX.data_ptr(), SX.data_ptr(), QW.data_ptr(), SW.data_ptr(), M, N, K, Y.data_ptr(), dtype, ws, bytes, stream));
    });
    return Y;
}

// nn.Linear4.forward
Tensor linear4_packed_weight(const Tensor &x, const Tensor &QW, const Tensor &SW, int N, int K)
{
    TORCH_CHECK(x.dim() >= 1 && x.size(-1) == K && x.numel() > 0, "input must be (..., ", K, ") and not empty, got ", x.sizes());
    no_tangent({&x});
    TORCH_CHECK(!wants_gradient({&x}), "a packed weight is for inference: take nn.linear8 for training");
    const Tensor x2 = matrix(x);
    auto shape = x.sizes().vec();
    shape.back() = N;
    return TAB_Linear4(x2, QW, SW, as_size(x2.size(0), "rows of the input"), N, K).view(shape);
}

// ---- router -----------------------------------------------------------------------------------------------------------

// [weights, experts, rows, places, offsets]
std::vector<Tensor> TAB_Route(const Tensor &logits, int M, int E, int k, bool normalize)
{
    const int dtype = dtype_code(logits.scalar_type(), "logits");
    TORCH_CHECK(M > 0 && E > 0, "M and E must be positive");
    TORCH_CHECK(k > 0 && k <= E, "k must be from 1 to E = ", E, ", got ", k);
    const int64_t ld = row_stride(logits, M, E, logits, "logits");
    const c10::hip::OptionalHIPGuardMasqueradingAsCUDA guard(logits.device());
    auto weights = device_empty({M, k}, torch::kFloat32, logits), experts = device_empty({M, k}, torch::kInt32, logits),
         rows = device_empty({(int64_t)M * k}, torch::kInt32, logits), places = device_empty({M, k}, torch::kInt32, logits),
         offsets = device_empty({E + 1}, torch::kInt32, logits);
    const size_t bytes = tab_route_workspace_bytes(M, E, k);
    with_workspace(bytes, logits, [&](void *ws, hipStream_t stream) {
        check_status(tab_route(logits.data_ptr(), dtype, (long)ld, M, E, k, normalize, weights.data_ptr<float>(), experts.data_ptr<int>(), rows.data_ptr<int>(),
                               places.data_ptr<int>(), offsets.data_ptr<int>(), ws, bytes, stream));
    });
    return {weights, experts, rows, places, offsets};
}

Tensor TAB_RouteBackward(const Tensor &dweights, const Tensor &weights, const Tensor &experts, const Tensor &logits, int M, int E, int k, bool normalize)
{
    const int dtype = dtype_code(logits.scalar_type(), "logits");
    TORCH_CHECK(M > 0 && E > 0, "M and E must be positive");
    TORCH_CHECK(k > 0 && k <= E, "k must be from 1 to E = ", E, ", got ", k);
    const int64_t ld = row_stride(logits, M, E, logits, "logits"), count = (int64_t)M * k;
    check_whole(dweights, count, torch::kFloat32, logits, "dweights");
    check_whole(weights, count, torch::kFloat32, logits, "weights");
    const int *chosen = int32s(experts, count, logits, "experts");
    const c10::hip::OptionalHIPGuardMasqueradingAsCUDA guard(logits.device());
    auto out = device_empty({M, E}, logits.scalar_type(), logits);
    check_status(tab_route_backward(dweights.data_ptr<float>(), weights.data_ptr<float>(), chosen, logits.data_ptr(), dtype, (long)ld, M, E, k, normalize, out.data_ptr(),
                                    current_stream(logits)));
    return out;
}

// ---- products over experts --------------------------------------------------------------------------------------------

// E weights of N x K packed one by one: [Q, S], of 8 bits with `transposed` [Q, S, QT, ST]
std::vector<Tensor> TAB_QuantizeExperts(const Tensor &W, int E, int N, int K, int bits, bool transposed)
{
    TORCH_CHECK(bits == 4 || bits == 8, "bits must be 4 or 8, got ", bits);
    TORCH_CHECK(bits == 8 || !transposed, "weights of 4 bits are not packed transposed");
    if (bits == 4) return quantize4(W, E, N, K, true);
    const int dtype = dtype_code(W.scalar_type(), "W");
    TORCH_CHECK(E > 0 && N > 0 && K > 0, "E, N and K must be positive");
    const int64_t ld = row_stride(W, (int64_t)E * N, K, W, "W"), KB = padded(K) / 128, NB = padded(N) / 128;
    const c10::hip::OptionalHIPGuardMasqueradingAsCUDA guard(W.device());
    auto Q = device_empty({E, N, padded(K)}, torch::kFloat8_e4m3fn, W), S = device_empty({E, KB, NB}, kScaleType, W);
    Tensor QT, ST;
    if (transposed) {
        QT = device_empty({E, K, padded(N)}, torch::kFloat8_e4m3fn, W);
        ST = device_empty({E, NB, KB}, kScaleType, W);
    }
    check_status(tab_quantize8_experts(W.data_ptr(), dtype, E, N, K, (long)ld, Q.data_ptr(), S.data_ptr(), data(QT), data(ST), current_stream(W)));
    if (transposed) return {Q, S, QT, ST};
    return {Q, S};
}

struct ExpertWeight { int bits, block_rows; };

ExpertWeight check_experts_weight(const Tensor &QW, const Tensor &SW, int64_t E, int N, int K, const Tensor &like)
{
    TORCH_CHECK(E > 0 && N > 0 && K > 0, "E, N and K must be positive");
    if (QW.scalar_type() == kFourBits) {
        check_weight4(QW, SW, E, N, K, like);
        return {4, 1};
    }
    check_whole(QW, E * N * padded(K), torch::kFloat8_e4m3fn, like, "QW");
    check_device(SW, like, "SW");
    const int64_t KB = padded(K) / 128;
    const int block_rows = SW.numel() == E * KB * N ? 1 : 128;
    check_whole(SW, block_rows == 1 ? E * KB * N : E * KB * (padded(N) / 128), kScaleType, like, "SW");
    return {8, block_rows};
}

void check_rows_of(const OptionalTensor &rows, int M, int R) { TORCH_CHECK(M > 0 && R > 0 && (rows || M == R), "without rows X has R = ", R, " rows, got M = ", M); }

Tensor TAB_ExpertsLinear(const Tensor &X, const OptionalTensor &rows, const Tensor &offsets, const Tensor &QW, const Tensor &SW, int M, int R, int E, int N, int K)
{
    const int dtype = dtype_code(X.scalar_type(), "X");
    check_rows_of(rows, M, R);
    const ExpertWeight w = check_experts_weight(QW, SW, E, N, K, X);
    const int64_t ld = row_stride(X, M, K, X, "X");
    const int *from = int32s(rows, R, X, "rows"), *at = int32s(offsets, E + 1, X, "offsets");
    const c10::hip::OptionalHIPGuardMasqueradingAsCUDA guard(X.device());
    auto Y = device_empty({R, N}, X.scalar_type(), X);
    const size_t bytes = tab_experts_linear_workspace_bytes(dtype, w.bits, M, R, E, N, K);
    with_workspace(bytes, X, [&](void *ws, hipStream_t stream) {
        check_status(tab_experts_linear(X.data_ptr(), dtype, (long)ld, M, from, at, QW.data_ptr(), SW.data_ptr(), w.bits, w.block_rows, R, E, N, K, Y.data_ptr(), ws, bytes, stream));
    });
    return Y;
}

Tensor experts_packed(const Tensor &QX, const Tensor &SX, const OptionalTensor &rows, const Tensor &offsets, const Tensor &QW, const Tensor &SW, int M, int R, int E, int N,
                      int K, torch::ScalarType out_type, bool full_sums)
{
    const int dtype = dtype_code(out_type, "the output"), format = format_of(QX, "QX");
    check_rows_of(rows, M, R);
    const ExpertWeight w = check_experts_weight(QW, SW, E, N, K, QX);
    check_whole(QX, M * padded(K), QX.scalar_type(), QX, "QX");
    check_whole(SX, M * (padded(K) / 128), kScaleType, QX, "SX");
    const int *from = int32s(rows, R, QX, "rows"), *at = int32s(offsets, E + 1, QX, "offsets");
    const c10::hip::OptionalHIPGuardMasqueradingAsCUDA guard(QX.device());
    auto Y = device_empty({R, N}, out_type, QX);
    const size_t bytes = tab_experts_linear_packed_workspace_bytes(dtype, full_sums, w.bits, R, E, N, K);
    with_workspace(bytes, QX, [&](void *ws, hipStream_t stream) {
        check_status(tab_experts_linear_packed(QX.data_ptr(), format, SX.data_ptr(), M, from, at, QW.data_ptr(), SW.data_ptr(), w.bits, w.block_rows, R, E, N, K, Y.data_ptr(),
                                               dtype, full_sums, ws, bytes, stream));
    });
    return Y;
}

// [QT, ST], with `sorted` [Q, S, QT, ST]
std::vector<Tensor> TAB_Quantize8ByExpert(const Tensor &X, const OptionalTensor &rows, const Tensor &offsets, int M, int R, int E, int K, int format, bool sorted)
{
    const int dtype = dtype_code(X.scalar_type(), "X");
    check_rows_of(rows, M, R);
    TORCH_CHECK(E > 0 && K > 0, "E and K must be positive");
    const int64_t ld = row_stride(X, M, K, X, "X");
    const int *from = int32s(rows, R, X, "rows"), *at = int32s(offsets, E + 1, X, "offsets");
    const c10::hip::OptionalHIPGuardMasqueradingAsCUDA guard(X.device());
    std::array<Tensor, 2> q;
    if (sorted) q = packed_empty(R, K, 1, format, X);
    const int64_t blocks = tab_run_blocks(R, E);
    auto QT = device_empty({K, 128 * blocks}, format_type(format), X), ST = device_empty({blocks, K}, kScaleType, X);
    check_status(tab_quantize8_by_expert(X.data_ptr(), dtype, (long)ld, M, from, at, R, E, K, format, data(q[0]), data(q[1]), QT.data_ptr(), ST.data_ptr(), current_stream(X)));
    if (sorted) return {q[0], q[1], QT, ST};
    return {QT, ST};
}

Tensor TAB_ExpertsGradWeight(const Tensor &QD, const Tensor &SD, const Tensor &QX, const Tensor &SX, const Tensor &offsets, int R, int E, int N, int K,
                             torch::ScalarType out_type)
{
    const int dtype = dtype_code(out_type, "the output"), format = format_of(QD, "QD");
    TORCH_CHECK(R > 0 && E > 0 && N > 0 && K > 0, "R, E, N and K must be positive");
    const int64_t blocks = tab_run_blocks(R, E);
    check_whole(QD, N * blocks * 128, QD.scalar_type(), QD, "QD");
    check_whole(SD, N * blocks, kScaleType, QD, "SD");
    check_whole(QX, K * blocks * 128, torch::kFloat8_e4m3fn, QD, "QX");
    check_whole(SX, K * blocks, kScaleType, QD, "SX");
    const int *at = int32s(offsets, E + 1, QD, "offsets");
    const c10::hip::OptionalHIPGuardMasqueradingAsCUDA guard(QD.device());
    auto dW = device_empty({E, N, K}, out_type, QD);
    check_status(tab_experts_grad_weight(QD.data_ptr(), format, SD.data_ptr(), QX.data_ptr(), SX.data_ptr(), at, R, E, N, K, dW.data_ptr(), dtype, current_stream(QD)));
    return dW;
}

// ---- back to the tokens -----------------------------------------------------------------------------------------------

Tensor combine_rows(const Tensor &Y, const Tensor &places, const OptionalTensor &weights, int M, int k, int R, int D, torch::ScalarType out_type)
{
    const int dtype = dtype_code(Y.scalar_type(), "Y"), out_dtype = dtype_code(out_type, "the output");
    TORCH_CHECK(M > 0 && k > 0 && R > 0 && D > 0, "M, k, R and D must be positive");
    check_whole(Y, (int64_t)R * D, Y.scalar_type(), Y, "Y");
    const int *at = int32s(places, (int64_t)M * k, Y, "places");
    if (weights) check_whole(*weights, (int64_t)M * k, torch::kFloat32, Y, "weights");
    const c10::hip::OptionalHIPGuardMasqueradingAsCUDA guard(Y.device());
    auto out = device_empty({M, D}, out_type, Y);
    check_status(tab_combine(Y.data_ptr(), dtype, at, weights ? weights->data_ptr<float>() : nullptr, M, k, R, D, out.data_ptr(), out_dtype, current_stream(Y)));
    return out;
}

Tensor TAB_Combine(const Tensor &Y, const Tensor &places, const OptionalTensor &weights, int M, int k, int R, int D)
{
    return combine_rows(Y, places, weights, M, k, R, D, Y.scalar_type());
}

// {dY, dweights}
std::vector<OptionalTensor> combine_backward(const Tensor &dout, const Tensor &Y, const Tensor &places, const OptionalTensor &weights, const OptionalTensor &offsets, int M,
                                             int k, int R, int D, bool want_dy, bool want_dweights)
{
    const int dtype = dtype_code(Y.scalar_type(), "Y");
    TORCH_CHECK(M > 0 && k > 0 && R > 0 && D > 0, "M, k, R and D must be positive");
    check_whole(Y, (int64_t)R * D, Y.scalar_type(), Y, "Y");
    check_whole(dout, (int64_t)M * D, Y.scalar_type(), Y, "dout");
    const int *at = int32s(places, (int64_t)M * k, Y, "places");
    if (weights) check_whole(*weights, (int64_t)M * k, torch::kFloat32, Y, "weights");
    TORCH_CHECK(!offsets || offsets->numel() > 1, "offsets must have E + 1 elements");
    const int *ends = offsets ? int32s(*offsets, offsets->numel(), Y, "offsets") + offsets->numel() - 1 : nullptr;
    const c10::hip::OptionalHIPGuardMasqueradingAsCUDA guard(Y.device());
    std::vector<OptionalTensor> out(2);
    if (want_dy) out[0] = device_empty({R, D}, Y.scalar_type(), Y);
    if (want_dweights) out[1] = device_empty({M, k}, torch::kFloat32, Y);
    check_status(tab_combine_backward(dout.data_ptr(), Y.data_ptr(), dtype, at, weights ? weights->data_ptr<float>() : nullptr, ends, M, k, R, D,
                                      out[0] ? out[0]->data_ptr() : nullptr, out[1] ? out[1]->data_ptr<float>() : nullptr, current_stream(Y)));
    return out;
}

std::vector<OptionalTensor> TAB_CombineBackward(const Tensor &dout, const Tensor &Y, const Tensor &places, const OptionalTensor &weights, const OptionalTensor &offsets,
                                                int M, int k, int R, int D)
{
    return combine_backward(dout, Y, places, weights, offsets, M, k, R, D, true, (bool)weights);
}

// ---- autograd ---------------------------------------------------------------------------------------------------------

struct RouteFunction : torch::autograd::Function<RouteFunction> {
    static torch::autograd::variable_list forward(torch::autograd::AutogradContext *ctx, const Tensor &logits, int64_t k, bool normalize)
    {
        const Tensor l2 = matrix(logits);
        const int M = as_size(l2.size(0), "tokens"), E = as_size(l2.size(1), "experts");
        auto out = TAB_Route(l2, M, E, (int)k, normalize);
        ctx->save_for_backward({l2, out[0], out[1]});
        ctx->saved_data["normalize"] = normalize;
        ctx->saved_data["shape"] = logits.sizes().vec();
        ctx->mark_non_differentiable({out[1], out[2], out[3], out[4]});
        ctx->set_materialize_grads(false);  // (zeros for the whole numbers would be four launches)
        return out;
    }
    static torch::autograd::variable_list backward(torch::autograd::AutogradContext *ctx, const torch::autograd::variable_list &grads)
    {
        no_second_derivative(grads);
        if (!grads[0].defined()) return {Tensor(), Tensor(), Tensor()};
        const auto saved = ctx->get_saved_variables();
        const Tensor &logits = saved[0];
        const int M = (int)logits.size(0), E = (int)logits.size(1), k = (int)saved[1].size(1);
        const Tensor d = TAB_RouteBackward(grads[0].contiguous(), saved[1], saved[2], logits, M, E, k, ctx->saved_data["normalize"].toBool());
        return {d.view(ctx->saved_data["shape"].toIntVector()), Tensor(), Tensor()};
    }
};

// nn.route
std::vector<Tensor> route(const Tensor &logits, int k, bool normalize)
{
    dtype_code(logits.scalar_type(), "logits");
    TORCH_CHECK(logits.dim() >= 1 && logits.numel() > 0, "logits must not be empty, got ", logits.sizes());
    no_tangent({&logits});
    if (wants_gradient({&logits})) return RouteFunction::apply(logits, (int64_t)k, normalize);
    const Tensor l2 = matrix(logits);
    return TAB_Route(l2, as_size(l2.size(0), "tokens"), as_size(l2.size(1), "experts"), k, normalize);
}

// The numbers of rows that a routing and an input agree in
struct Sizes {
    int M, R, E, k;
    Sizes(const Tensor &x, const Tensor &rows, const Tensor &places, const Tensor &offsets, int64_t E_, bool gather)
    {
        TORCH_CHECK(x.dim() >= 1 && x.numel() > 0, "x must not be empty, got ", x.sizes());
        TORCH_CHECK(places.dim() == 2 && places.numel() > 0 && rows.numel() == places.numel(), "places (M, k) and rows (M * k) must agree, got ", places.sizes(), " and ", rows.sizes());
        M = as_size(x.numel() / x.size(-1), "rows of x");
        R = as_size(rows.numel(), "rows");
        E = as_size(E_, "experts");
        k = (int)places.size(1);
        TORCH_CHECK(offsets.numel() == E_ + 1, "the routing is one of ", offsets.numel() - 1, " experts, the weights are ", E_);
        TORCH_CHECK(M == (gather ? places.size(0) : R), "x has ", M, " rows, the routing ", gather ? places.size(0) : R, gather ? " tokens" : " sorted rows");
    }
};

// y[r] = Q(x[rows[r]]) Q(w[e])^T, dx[t] = sum over t's rows of Q(dy[r]) Q(w[e]), dw[e] = Q(dy_e^T) Q(x_e^T)^T: three products of packed operands, all
// packed in the forward pass but dy.
struct ExpertsFunction : torch::autograd::Function<ExpertsFunction> {
    static Tensor forward(torch::autograd::AutogradContext *ctx, const Tensor &x, const Tensor &w, const Tensor &rows, const Tensor &places, const Tensor &offsets,
                          bool gather, int64_t grad_format)
    {
        const c10::hip::OptionalHIPGuardMasqueradingAsCUDA guard(x.device());
        const bool need_dx = x.requires_grad(), need_dw = w.requires_grad();
        const Tensor x2 = matrix(x), w2 = w.contiguous();
        const int K = as_size(x2.size(1), "columns of x"), N = as_size(w.size(1), "rows of an expert's weight");
        const Sizes s(x, rows, places, offsets, w.size(0), gather);
        // what the backward pass would refuse is refused here
        check_status(tab_experts_check_gradients(dtype_code(x.scalar_type(), "x"), dtype_code(w.scalar_type(), "w"), s.M, gather ? s.k : 0, s.R, s.E, N, K, need_dx, need_dw));
        const auto from = gather ? OptionalTensor(rows) : c10::nullopt;
        Tensor q, sx, qt, st;
        if (need_dw) {
            const auto packed = TAB_Quantize8ByExpert(x2, from, offsets, s.M, s.R, s.E, K, TAB_E4M3, !gather);
            qt = packed[gather ? 0 : 2], st = packed[gather ? 1 : 3];
            if (!gather) q = packed[0], sx = packed[1];
        }
        if (!q.defined()) {
            auto packed = packed_empty(s.M, K, 1, TAB_E4M3, x2);
            q = packed[0], sx = packed[1];
            check_status(tab_quantize8(x2.data_ptr(), dtype_code(x2.scalar_type(), "x"), s.M, K, (long)row_stride(x2, s.M, K, x2, "x"), 1, TAB_E4M3, q.data_ptr(),
                                       sx.data_ptr(), nullptr, nullptr, current_stream(x2)));
        }
        const auto qw = TAB_QuantizeExperts(w2, s.E, N, K, 8, need_dx);
        Tensor y = experts_packed(q, sx, from, offsets, qw[0], qw[1], s.M, s.R, s.E, N, K, x.scalar_type(), true);
        ctx->save_for_backward({qt, st, need_dx ? qw[2] : Tensor(), need_dx ? qw[3] : Tensor(), offsets, places});
        ctx->saved_data["sizes"] = std::vector<int64_t>{s.M, s.R, s.E, s.k, N, K, gather, grad_format, (int64_t)x.scalar_type(), (int64_t)w.scalar_type()};
        ctx->saved_data["shape"] = x.sizes().vec();
        return y;
    }
    static torch::autograd::variable_list backward(torch::autograd::AutogradContext *ctx, const torch::autograd::variable_list &grads)
    {
        no_second_derivative(grads);
        const auto saved = ctx->get_saved_variables();
        const auto sizes = ctx->saved_data["sizes"].toIntVector();
        const int M = (int)sizes[0], R = (int)sizes[1], E = (int)sizes[2], k = (int)sizes[3], N = (int)sizes[4], K = (int)sizes[5], format = (int)sizes[7];
        const bool gather = sizes[6] != 0, need_dw = saved[0].defined(), need_dx = saved[2].defined();
        const auto x_type = (torch::ScalarType)sizes[8], w_type = (torch::ScalarType)sizes[9];
        const Tensor dy = matrix(grads[0]), &offsets = saved[4];
        const c10::hip::OptionalHIPGuardMasqueradingAsCUDA guard(dy.device());
        Tensor q, s, qt, st, dx, dw;
        if (need_dw) {
            const auto packed = TAB_Quantize8ByExpert(dy, c10::nullopt, offsets, R, R, E, N, format, need_dx);
            qt = packed[need_dx ? 2 : 0], st = packed[need_dx ? 3 : 1];
            if (need_dx) q = packed[0], s = packed[1];
        } else if (need_dx) {
            auto packed = packed_empty(R, N, 1, format, dy);
            q = packed[0], s = packed[1];
            check_status(tab_quantize8(dy.data_ptr(), dtype_code(dy.scalar_type(), "dy"), R, N, (long)row_stride(dy, R, N, dy, "dy"), 1, format, q.data_ptr(), s.data_ptr(),
                                       nullptr, nullptr, current_stream(dy)));
        }
        if (need_dx) {
            // the rows of a token in fp32, added up and rounded once
            const Tensor rows = experts_packed(q, s, c10::nullopt, offsets, saved[2], saved[3], R, R, E, K, N, gather ? torch::kFloat32 : x_type, x_type == torch::kFloat32);
            dx = (gather ? combine_rows(rows, saved[5], c10::nullopt, M, k, R, K, x_type) : rows).view(ctx->saved_data["shape"].toIntVector());
        }
        if (need_dw) dw = TAB_ExpertsGradWeight(qt, st, saved[0], saved[1], offsets, R, E, N, K, w_type);
        return {dx, dw, Tensor(), Tensor(), Tensor(), Tensor(), Tensor()};
    }
};

// nn.experts_linear8
Tensor experts_linear8(const Tensor &x, const Tensor &w, const Tensor &rows, const Tensor &places, const Tensor &offsets, bool gather, int grad_format)
{
    dtype_code(x.scalar_type(), "x");
    dtype_code(w.scalar_type(), "w");
    format_type(grad_format);
    TORCH_CHECK(x.dim() >= 1 && w.dim() == 3 && x.size(-1) == w.size(2), "x (..., K) and w (E, N, K) must agree in K, got ", x.sizes(), " and ", w.sizes());
    TORCH_CHECK(w.numel() > 0, "w must not be empty, got ", w.sizes());
    no_tangent({&x, &w});
    const Sizes s(x, rows, places, offsets, w.size(0), gather);
    check_device(w, x, "w");
    int32s(places, s.R, x, "places");  // (of the backward pass alone)
    if (wants_gradient({&x, &w})) return ExpertsFunction::apply(x, w, rows, places, offsets, gather, (int64_t)grad_format);
    const Tensor x2 = matrix(x), w2 = w.contiguous();
    const int K = as_size(x2.size(1), "columns of x"), N = as_size(w.size(1), "rows of an expert's weight");
    const c10::hip::OptionalHIPGuardMasqueradingAsCUDA guard(x.device());
    const auto qw = TAB_QuantizeExperts(w2, s.E, N, K, 8, false);
    return TAB_ExpertsLinear(x2, gather ? OptionalTensor(rows) : c10::nullopt, offsets, qw[0], qw[1], s.M, s.R, s.E, N, K);
}

// nn.PackedExperts.forward
Tensor experts_packed_weight(const Tensor &x, const Tensor &QW, const Tensor &SW, const Tensor &rows, const Tensor &places, const Tensor &offsets, bool gather, int E, int N,
                             int K)
{
    TORCH_CHECK(x.dim() >= 1 && x.size(-1) == K && x.numel() > 0, "input must be (..., ", K, ") and not empty, got ", x.sizes());
    no_tangent({&x});
    TORCH_CHECK(!wants_gradient({&x}), "packed weights are for inference: take nn.experts_linear8 for training");
    const Sizes s(x, rows, places, offsets, E, gather);
    return TAB_ExpertsLinear(matrix(x), gather ? OptionalTensor(rows) : c10::nullopt, offsets, QW, SW, s.M, s.R, E, N, K);
}

struct CombineFunction : torch::autograd::Function<CombineFunction> {
    static Tensor forward(torch::autograd::AutogradContext *ctx, const Tensor &y, const Tensor &weights, const Tensor &places, const Tensor &offsets)
    {
        const Tensor y2 = y.contiguous(), w2 = weights.contiguous();
        const int M = as_size(places.size(0), "tokens"), k = as_size(places.size(1), "choices"), R = as_size(y.size(0), "rows of y"), D = as_size(y.size(1), "columns of y");
        ctx->save_for_backward({y2, w2, places, offsets});
        ctx->saved_data["wanted"] = std::vector<int64_t>{y.requires_grad(), weights.requires_grad()};
        return TAB_Combine(y2, places, w2, M, k, R, D);
    }
    static torch::autograd::variable_list backward(torch::autograd::AutogradContext *ctx, const torch::autograd::variable_list &grads)
    {
        no_second_derivative(grads);
        const auto saved = ctx->get_saved_variables();
        const auto wanted = ctx->saved_data["wanted"].toIntVector();
        const Tensor &y = saved[0], &places = saved[2];
        const auto out = combine_backward(grads[0].contiguous(), y, places, saved[1], saved[3], (int)places.size(0), (int)places.size(1), (int)y.size(0), (int)y.size(1),
                                          wanted[0] != 0, wanted[1] != 0);
        return {out[0] ? *out[0] : Tensor(), out[1] ? *out[1] : Tensor(), Tensor(), Tensor()};
    }
};

// nn.combine
Tensor combine(const Tensor &y, const Tensor &any_weights, const Tensor &places, const Tensor &offsets)
{
    dtype_code(y.scalar_type(), "y");
    TORCH_CHECK(y.dim() == 2 && y.numel() > 0, "y must be (rows, D) and not empty, got ", y.sizes());
    TORCH_CHECK(places.dim() == 2 && places.numel() == y.size(0) && any_weights.sizes() == places.sizes(), "places and weights must be (M, k) with M * k = ", y.size(0),
                " rows of y, got ", places.sizes(), " and ", any_weights.sizes());
    no_tangent({&y, &any_weights});
    check_device(any_weights, y, "weights");
    const auto type = any_weights.scalar_type();
    const Tensor weights = type == torch::kBFloat16 || type == torch::kFloat16 ? any_weights.to(torch::kFloat32) : any_weights;
    TORCH_CHECK(offsets.numel() > 1, "offsets must have E + 1 elements");
    int32s(offsets, offsets.numel(), y, "offsets");
    if (wants_gradient({&y, &weights})) return CombineFunction::apply(y, weights, places, offsets);
    return TAB_Combine(y.contiguous(), places, weights.contiguous(), as_size(places.size(0), "tokens"), as_size(places.size(1), "choices"), as_size(y.size(0), "rows of y"),
                       as_size(y.size(1), "columns of y"));
}

}  // namespace

void bind_experts(pybind11::module_ &m)
{
    using pybind11::arg;
    m.def("Quantize4", &TAB_Quantize4, "X packed in 4 bits with a power-of-two scale per group of 32: [Q, S]", arg("X"), arg("M"), arg("K"));
    m.def("Linear4", &TAB_Linear4, "X, quantized on the way, times packed weights of 4 bits", arg("X"), arg("QW"), arg("SW"), arg("M"), arg("N"), arg("K"));
    m.def(
        "Linear4Packed",
        [](const Tensor &QX, const Tensor &SX, const Tensor &QW, const Tensor &SW, int M, int N, int K, const pybind11::object &out_dtype) {
            return TAB_Linear4Packed(QX, SX, QW, SW, M, N, K, scalar_type(out_dtype));
        },
        "Product of a packed activation and packed weights of 4 bits");
    m.def("linear4_packed_weight", &linear4_packed_weight, "nn.Linear4.forward");
    m.def("Route", &TAB_Route, "the k best experts of each token and the rows in their order: [weights, experts, rows, places, offsets]");
    m.def("RouteBackward", &TAB_RouteBackward, "gradient of Route's weights");
    m.def("QuantizeExperts", &TAB_QuantizeExperts, "weights of experts packed one by one");
    m.def("ExpertsLinear", &TAB_ExpertsLinear, "rows sorted by expert times their expert's packed weight");
    m.def(
        "ExpertsLinearPacked",
        [](const Tensor &QX, const Tensor &SX, const OptionalTensor &rows, const Tensor &offsets, const Tensor &QW, const Tensor &SW, int M, int R, int E, int N, int K,
           const pybind11::object &out_dtype) { return experts_packed(QX, SX, rows, offsets, QW, SW, M, R, E, N, K, scalar_type(out_dtype), true); },
        "ExpertsLinear on a packed activation");
    m.def("Quantize8ByExpert", &TAB_Quantize8ByExpert, "rows sorted by expert, packed for the gradients of the weights");
    m.def(
        "ExpertsGradWeight",
        [](const Tensor &QD, const Tensor &SD, const Tensor &QX, const Tensor &SX, const Tensor &offsets, int R, int E, int N, int K, const pybind11::object &out_dtype) {
            return TAB_ExpertsGradWeight(QD, SD, QX, SX, offsets, R, E, N, K, scalar_type(out_dtype));
        },
        "gradients of the experts' weights");
    m.def("Combine", &TAB_Combine, "the experts' rows back to their tokens");
    m.def("CombineBackward", &TAB_CombineBackward, "gradients of Combine");
    m.def("route", &route, "nn.route");
    m.def("experts_linear8", &experts_linear8, "nn.experts_linear8");
    m.def("experts_packed_weight", &experts_packed_weight, "nn.PackedExperts.forward");
    m.def("combine", &combine, "nn.combine");
}
