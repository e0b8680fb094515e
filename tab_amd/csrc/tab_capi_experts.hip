// C ABI of the 4-bit layers and of layers of experts: argument checks and launches.  No allocation, no synchronisation, no host<->device copy.
#include "tab_checks8.h"
#include "tab_experts.h"

namespace {

int check_matrices(int E, int M, int K, long threads)
{
    if (E < 1 || M < 1 || K < 1) return fail(TAB_ERR_BAD_ARGUMENT, "E, M and K must be positive");
    if ((long)E * M > kMostRows || threads > kMostThreads) return fail(TAB_ERR_BAD_SHAPE, "matrix too large for one launch");
    return TAB_OK;
}

int check_int32(const void *p, const char *what, bool optional = false)
{
    if (!p && !optional) return fail(TAB_ERR_BAD_ARGUMENT, "null device pointer: %s", what);
    return (uintptr_t)p % 4 ? fail(TAB_ERR_BAD_ARGUMENT, "%s must be aligned to its elements", what) : TAB_OK;
}

int check_weight_bits(int bits, int w_block_rows)
{
    if (bits != 4 && bits != 8) return fail(TAB_ERR_BAD_ARGUMENT, "weights must have 4 or 8 bits, got %d", bits);
    if (bits == 8) return check_block_rows(w_block_rows);
    return TAB_OK;
}

// Columns of a product with weights of 4 bits
int check_columns4(int N)
{
    return N > tab::kRows4Most ? fail(TAB_ERR_BAD_SHAPE, "weights of 4 bits may have %d rows, got %d: their scales are found by 32-bit offsets", tab::kRows4Most, N) : TAB_OK;
}

// Rows sorted by expert: the sizes of what is done with them, then the operands
int check_run_sizes(int M, int R, int E)
{
    if (M < 1 || R < 1) return fail(TAB_ERR_BAD_ARGUMENT, "M and R must be positive");
    if (E < 1 || E > tab::kExpertsMost) return fail(TAB_ERR_BAD_ARGUMENT, "there must be 1 to %d experts, got %d", tab::kExpertsMost, E);
    if (M > kMostRows || R > kMostRows) return fail(TAB_ERR_BAD_SHAPE, "too many rows: %d and %d", M, R);
    return TAB_OK;
}

int check_runs(int M, const int *rows, const int *offsets, int R, int E)
{
    TAB_CHECK(check_run_sizes(M, R, E));
    TAB_CHECK(check_int32(rows, "rows", true));
    TAB_CHECK(check_int32(offsets, "offsets"));
    if (!rows && M != R) return fail(TAB_ERR_BAD_ARGUMENT, "without rows X has the R = %d rows of Y, got %d", R, M);
    return TAB_OK;
}

int check_experts_sizes(int M, bool listed, int R, int E, int N, int K, int out_dtype, bool full_sums, int w_bits)
{
    TAB_CHECK(check_run_sizes(M, R, E));
    if (N < 1 || K < 1) return fail(TAB_ERR_BAD_ARGUMENT, "N and K must be positive");
    const int KB = tab::blocks8(K);
    if (N > kMostRows || KB > tab::kBlocks8Most) return fail(TAB_ERR_BAD_SHAPE, "product too large for 32-bit offsets into a tile");
    if (w_bits == 4) TAB_CHECK(check_columns4(N));
    const tab::ExpertsPlan plan = tab::experts_plan(out_dtype, full_sums, w_bits, R, E, N, KB);
    if (plan.workgroups * 512 > kMostThreads) return fail(TAB_ERR_BAD_SHAPE, "product too large for one launch");
    // listed rows are read by 32-bit offsets into all of X, rows as they are sorted by those into a tile
    if (!plan.few && listed && (unsigned long)M * (unsigned long)KB * tab::kBlock8 > 0xe0000000ul)
        return fail(TAB_ERR_BAD_SHAPE, "X takes more than 3.5 GiB packed: too large for the 32-bit offsets of listed rows");
    return TAB_OK;
}

int check_experts(int M, const int *rows, const int *offsets, int R, int E, int N, int K, int out_dtype, bool full_sums, int w_bits, int w_block_rows)
{
    TAB_CHECK(check_type(out_dtype, "out_dtype"));
    TAB_CHECK(check_weight_bits(w_bits, w_block_rows));
    TAB_CHECK(check_runs(M, rows, offsets, R, E));
    return check_experts_sizes(M, rows != nullptr, R, E, N, K, out_dtype, full_sums, w_bits);
}

int check_by_expert_sizes(int M, int R, int E, int K)
{
    TAB_CHECK(check_run_sizes(M, R, E));
    if (K < 1) return fail(TAB_ERR_BAD_ARGUMENT, "K must be positive");
    if ((long)tab::run_blocks_most(R, E) * tab::blocks8(K) * 256 > kMostThreads) return fail(TAB_ERR_BAD_SHAPE, "matrix too large for one launch");
    return TAB_OK;
}

int check_grad_sizes(int R, int E, int N, int K, int out_dtype)
{
    TAB_CHECK(check_run_sizes(R, R, E));
    if (N < 1 || K < 1) return fail(TAB_ERR_BAD_ARGUMENT, "N and K must be positive");
    if (N > kMostRows || K > kMostRows || tab::run_blocks_most(R, E) > tab::kBlocks8Most)
        return fail(TAB_ERR_BAD_SHAPE, "gradients of weights from more blocks of rows than %d: too large for 32-bit offsets into a tile", tab::kBlocks8Most);
    if (tab::experts_grad_workgroups(out_dtype, R, E, N, K) * 512 > kMostThreads) return fail(TAB_ERR_BAD_SHAPE, "product too large for one launch");
    return TAB_OK;
}

int check_combine_sizes(int M, int k, int R, int D)
{
    if (M < 1 || k < 1 || R < 1 || D < 1) return fail(TAB_ERR_BAD_ARGUMENT, "M, k, R and D must be positive");
    if ((long)M * k > kMostRows || R > kMostRows || D > kMostRows || (long)M * ((D + 7) / 8) > kMostRows || (long)M * 256 > kMostThreads)
        return fail(TAB_ERR_BAD_SHAPE, "too large for one launch");
    return TAB_OK;
}

// Weights of 4 bits have full sums towards fp32 in any case
bool full_sums_of(int full_sums, int w_bits) { return full_sums != 0 || w_bits == 4; }

size_t parts_bytes(const tab::ExpertsPlan &plan, int R, int N) { return plan.few || plan.parts == 1 ? 0 : (size_t)plan.parts * (size_t)R * (size_t)N * sizeof(float); }

tab::ExpertsArgs experts_args(const void *x, const void *sx, long ldx, int M, const int *rows, const int *offsets, const void *qw, const void *sw, int w_block_rows,
                              int R, int E, int N, int K, void *y)
{
    return {x, static_cast<const uint8_t *>(sx), static_cast<const uint8_t *>(qw), static_cast<const uint8_t *>(sw), y, offsets, rows, M, R, E, N, K, tab::blocks8(K),
            w_block_rows, ldx};
}

}  // namespace

extern "C" {

int tab_quantize4(const void *dev_W, int dtype, int E, int M, int K, long ldw, void *dev_Q, void *dev_S, void *stream)
{
    TAB_CHECK(check_type(dtype, "dtype"));
    TAB_CHECK(check_matrices(E, M, K, E < 1 || M < 1 || K < 1 ? 0 : tab::quantize4_tiles((long)E * M, K) * 256));
    TAB_CHECK(check_rows(dev_W, dtype, E * M, K, ldw, "W"));
    TAB_CHECK(check_packed(dev_Q, dev_S, "Q or S"));
    const tab::Quantize4Args a = {dev_W, static_cast<uint8_t *>(dev_Q), static_cast<uint8_t *>(dev_S), E, M, K, ldw};
    const hipError_t e = tab::launch_quantize4(dtype, a, static_cast<hipStream_t>(stream));
    return e == hipSuccess ? TAB_OK : device_fail(e, "quantize4 launch");
}

size_t tab_linear4_packed_workspace_bytes(int out_dtype, int M, int N, int K)
{
    return M < 1 || N < 1 || K < 1 ? 0 : tab::linear4_workspace(out_dtype, M, N, tab::blocks8(K));
}

int tab_linear4_packed(const void *dev_QX, const void *dev_SX, const void *dev_QW, const void *dev_SW, int M, int N, int K, void *dev_Y, int out_dtype,
                       void *workspace, size_t workspace_bytes, void *stream)
{
    TAB_CHECK(check_type(out_dtype, "out_dtype"));
    TAB_CHECK(check_linear(out_dtype, M, N, K));
    TAB_CHECK(check_columns4(N));
    TAB_CHECK(check_packed(dev_QX, dev_SX, "QX or SX"));
    TAB_CHECK(check_packed(dev_QW, dev_SW, "QW or SW"));
    if ((uintptr_t)dev_SW % 4) return fail(TAB_ERR_BAD_ARGUMENT, "SW must be aligned to 4 bytes");
    TAB_CHECK(check_rows(dev_Y, out_dtype, 1, N, N, "Y"));
    TAB_CHECK(check_workspace(workspace, workspace_bytes, tab_linear4_packed_workspace_bytes(out_dtype, M, N, K)));
    const tab::Linear8Args a = {static_cast<const uint8_t *>(dev_QX), static_cast<const uint8_t *>(dev_SX), static_cast<const uint8_t *>(dev_QW),
                                static_cast<const uint8_t *>(dev_SW), dev_Y, M, N, tab::blocks8(K), 1};
    const hipError_t e = tab::launch_linear4(out_dtype, a, workspace, static_cast<hipStream_t>(stream));
    return e == hipSuccess ? TAB_OK : device_fail(e, "linear4 launch");
}

size_t tab_linear4_workspace_bytes(int dtype, int M, int N, int K)
{
    if (M < 1 || N < 1 || K < 1 || tab::linear4_rows_supported(M, N, K)) return 0;
    return packed_bytes(M, K) + tab_linear4_packed_workspace_bytes(dtype, M, N, K);
}

int tab_linear4(const void *dev_X, int dtype, long ldx, const void *dev_QW, const void *dev_SW, int M, int N, int K, void *dev_Y, void *workspace,
                size_t workspace_bytes, void *stream)
{
    TAB_CHECK(check_type(dtype, "dtype"));
    TAB_CHECK(check_linear(dtype, M, N, K));
    TAB_CHECK(check_columns4(N));
    TAB_CHECK(check_rows(dev_X, dtype, M, K, ldx, "X"));
    TAB_CHECK(check_packed(dev_QW, dev_SW, "QW or SW"));
    if ((uintptr_t)dev_SW % 4) return fail(TAB_ERR_BAD_ARGUMENT, "SW must be aligned to 4 bytes");
    TAB_CHECK(check_rows(dev_Y, dtype, 1, N, N, "Y"));
    if (tab::linear4_rows_supported(M, N, K)) {
        const tab::Linear8RowsArgs a = {dev_X, static_cast<const uint8_t *>(dev_QW), static_cast<const uint8_t *>(dev_SW), dev_Y, M, N, K, 1, ldx};
        const hipError_t e = tab::launch_linear4_rows(dtype, a, static_cast<hipStream_t>(stream));
        return e == hipSuccess ? TAB_OK : device_fail(e, "linear4 launch");
    }
    TAB_CHECK(check_quantize(M, K, 1, false));
    TAB_CHECK(check_workspace(workspace, workspace_bytes, tab_linear4_workspace_bytes(dtype, M, N, K)));
    uint8_t *const q = static_cast<uint8_t *>(workspace), *const s = q + packed_numbers(M, K);
    const size_t packed = packed_bytes(M, K);
    TAB_CHECK(tab_quantize8(dev_X, dtype, M, K, ldx, 1, TAB_E4M3, q, s, nullptr, nullptr, stream));
    return tab_linear4_packed(q, s, dev_QW, dev_SW, M, N, K, dev_Y, dtype, q + packed, workspace_bytes - packed, stream);
}

size_t tab_route_workspace_bytes(int M, int E, int k) { return M < 1 || E < 1 || k < 1 || E > tab::kExpertsMost ? 0 : tab::route_workspace(M, E, k); }

static int check_route(const void *logits, int dtype, long ld, int M, int E, int k)
{
    TAB_CHECK(check_type(dtype, "dtype"));
    if (M < 1) return fail(TAB_ERR_BAD_ARGUMENT, "M must be positive");
    if (E < 1 || E > tab::kExpertsMost) return fail(TAB_ERR_BAD_ARGUMENT, "there must be 1 to %d experts, got %d", tab::kExpertsMost, E);
    if (k < 1 || k > E || k > tab::kChoicesMost) return fail(TAB_ERR_BAD_ARGUMENT, "k must be from 1 to E and to %d, got %d", tab::kChoicesMost, k);
    if ((long)M * k > kMostRows) return fail(TAB_ERR_BAD_SHAPE, "too many rows: %d tokens of %d", M, k);
    return check_rows(logits, dtype, M, E, ld, "logits");
}

int tab_route(const void *dev_logits, int dtype, long ld, int M, int E, int k, int normalize, float *dev_weights, int *dev_experts, int *dev_rows, int *dev_places,
              int *dev_offsets, void *workspace, size_t workspace_bytes, void *stream)
{
    TAB_CHECK(check_route(dev_logits, dtype, ld, M, E, k));
    TAB_CHECK(check_int32(dev_weights, "weights"));
    TAB_CHECK(check_int32(dev_experts, "experts"));
    TAB_CHECK(check_int32(dev_rows, "rows"));
    TAB_CHECK(check_int32(dev_places, "places"));
    TAB_CHECK(check_int32(dev_offsets, "offsets"));
    TAB_CHECK(check_workspace(workspace, workspace_bytes, tab_route_workspace_bytes(M, E, k)));
    const tab::RouteArgs a = {dev_logits, dev_weights, dev_experts, dev_rows, dev_places, dev_offsets, static_cast<int *>(workspace), ld, M, E, k, normalize != 0};
    const hipError_t e = tab::launch_route(dtype, a, static_cast<hipStream_t>(stream));
    return e == hipSuccess ? TAB_OK : device_fail(e, "route launch");
}

int tab_route_backward(const float *dev_dweights, const float *dev_weights, const int *dev_experts, const void *dev_logits, int dtype, long ld, int M, int E, int k,
                       int normalize, void *dev_dlogits, void *stream)
{
    TAB_CHECK(check_route(dev_logits, dtype, ld, M, E, k));
    TAB_CHECK(check_int32(dev_dweights, "dweights"));
    TAB_CHECK(check_int32(dev_weights, "weights"));
    TAB_CHECK(check_int32(dev_experts, "experts"));
    TAB_CHECK(check_rows(dev_dlogits, dtype, 1, E, E, "dlogits"));
    const tab::RouteGradArgs a = {dev_dweights, dev_weights, dev_experts, dev_logits, dev_dlogits, ld, M, E, k, normalize != 0};
    const hipError_t e = tab::launch_route_grad(dtype, a, static_cast<hipStream_t>(stream));
    return e == hipSuccess ? TAB_OK : device_fail(e, "route gradient launch");
}

int tab_run_blocks(int R, int E) { return R < 1 || E < 1 ? 0 : tab::run_blocks_most(R, E); }

int tab_quantize8_experts(const void *dev_W, int dtype, int E, int N, int K, long ldw, void *dev_Q, void *dev_S, void *dev_QT, void *dev_ST, void *stream)
{
    TAB_CHECK(check_type(dtype, "dtype"));
    TAB_CHECK(check_matrices(E, N, K, E < 1 || N < 1 || K < 1 ? 0 : tab::quantize8_tiles(tab::kBlock8, true, N, K) * 256 * E));
    if (E > tab::kExpertsMost) return fail(TAB_ERR_BAD_ARGUMENT, "there must be 1 to %d experts, got %d", tab::kExpertsMost, E);
    TAB_CHECK(check_rows(dev_W, dtype, E * N, K, ldw, "W"));
    if (!dev_Q && !dev_QT) return fail(TAB_ERR_BAD_ARGUMENT, "null device pointer: Q and QT");
    if (dev_Q || dev_S) TAB_CHECK(check_packed(dev_Q, dev_S, "Q or S"));
    if (dev_QT || dev_ST) TAB_CHECK(check_packed(dev_QT, dev_ST, "QT or ST"));
    const tab::Quantize8Args a = {dev_W, static_cast<uint8_t *>(dev_Q), static_cast<uint8_t *>(dev_S), static_cast<uint8_t *>(dev_QT), static_cast<uint8_t *>(dev_ST), N, K, ldw, E};
    const hipError_t e = tab::launch_quantize8(dtype, TAB_E4M3, tab::kBlock8, a, static_cast<hipStream_t>(stream));
    return e == hipSuccess ? TAB_OK : device_fail(e, "quantize8 launch");
}

int tab_quantize8_by_expert(const void *dev_X, int dtype, long ldx, int M, const int *dev_rows, const int *dev_offsets, int R, int E, int K, int format, void *dev_Q,
                            void *dev_S, void *dev_QT, void *dev_ST, void *stream)
{
    TAB_CHECK(check_type(dtype, "dtype"));
    TAB_CHECK(check_format(format));
    TAB_CHECK(check_runs(M, dev_rows, dev_offsets, R, E));
    TAB_CHECK(check_by_expert_sizes(M, R, E, K));
    TAB_CHECK(check_rows(dev_X, dtype, M, K, ldx, "X"));
    if (dev_Q || dev_S) TAB_CHECK(check_packed(dev_Q, dev_S, "Q or S"));
    TAB_CHECK(check_packed(dev_QT, dev_ST, "QT or ST"));
    const tab::Quantize8Args a = {dev_X, static_cast<uint8_t *>(dev_Q), static_cast<uint8_t *>(dev_S), static_cast<uint8_t *>(dev_QT), static_cast<uint8_t *>(dev_ST), R, K, ldx};
    const hipError_t e = tab::launch_quantize8_by_expert(dtype, format, a, dev_offsets, dev_rows, E, M, static_cast<hipStream_t>(stream));
    return e == hipSuccess ? TAB_OK : device_fail(e, "quantize8 launch");
}

size_t tab_experts_linear_packed_workspace_bytes(int out_dtype, int full_sums, int w_bits, int R, int E, int N, int K)
{
    return R < 1 || E < 1 || N < 1 || K < 1 ? 0 : parts_bytes(tab::experts_plan(out_dtype, full_sums_of(full_sums, w_bits), w_bits, R, E, N, tab::blocks8(K)), R, N);
}

int tab_experts_linear_packed(const void *dev_QX, int x_format, const void *dev_SX, int M, const int *dev_rows, const int *dev_offsets, const void *dev_QW,
                              const void *dev_SW, int w_bits, int w_block_rows, int R, int E, int N, int K, void *dev_Y, int out_dtype, int full_sums,
                              void *workspace, size_t workspace_bytes, void *stream)
{
    TAB_CHECK(check_format(x_format));
    TAB_CHECK(check_experts(M, dev_rows, dev_offsets, R, E, N, K, out_dtype, full_sums_of(full_sums, w_bits), w_bits, w_block_rows));
    if (w_bits == 4 && x_format != TAB_E4M3) return fail(TAB_ERR_BAD_ARGUMENT, "weights of 4 bits take activations in E4M3");
    TAB_CHECK(check_packed(dev_QX, dev_SX, "QX or SX"));
    TAB_CHECK(check_packed(dev_QW, dev_SW, "QW or SW"));
    if (w_bits == 4 && (uintptr_t)dev_SW % 4) return fail(TAB_ERR_BAD_ARGUMENT, "SW must be aligned to 4 bytes");
    TAB_CHECK(check_rows(dev_Y, out_dtype, 1, N, N, "Y"));
    TAB_CHECK(check_workspace(workspace, workspace_bytes, tab_experts_linear_packed_workspace_bytes(out_dtype, full_sums, w_bits, R, E, N, K)));
    const tab::ExpertsPlan plan = tab::experts_plan(out_dtype, full_sums_of(full_sums, w_bits), w_bits, R, E, N, tab::blocks8(K));
    const tab::ExpertsArgs a = experts_args(dev_QX, dev_SX, 0, M, dev_rows, dev_offsets, dev_QW, dev_SW, w_block_rows, R, E, N, K, dev_Y);
    const hipError_t e = w_bits == 4 ? tab::launch_experts4(out_dtype, plan, a, workspace, static_cast<hipStream_t>(stream))
                                     : tab::launch_experts8(out_dtype, full_sums != 0, x_format, plan, a, workspace, static_cast<hipStream_t>(stream));
    return e == hipSuccess ? TAB_OK : device_fail(e, "experts launch");
}

size_t tab_experts_linear_workspace_bytes(int dtype, int w_bits, int M, int R, int E, int N, int K)
{
    if (M < 1 || R < 1 || E < 1 || N < 1 || K < 1) return 0;
    const tab::ExpertsPlan plan = tab::experts_plan(dtype, true, w_bits, R, E, N, tab::blocks8(K));
    return plan.few ? 0 : packed_bytes(M, K) + parts_bytes(plan, R, N);
}

int tab_experts_linear(const void *dev_X, int dtype, long ldx, int M, const int *dev_rows, const int *dev_offsets, const void *dev_QW, const void *dev_SW, int w_bits,
                       int w_block_rows, int R, int E, int N, int K, void *dev_Y, void *workspace, size_t workspace_bytes, void *stream)
{
    TAB_CHECK(check_experts(M, dev_rows, dev_offsets, R, E, N, K, dtype, true, w_bits, w_block_rows));
    TAB_CHECK(check_rows(dev_X, dtype, M, K, ldx, "X"));
    TAB_CHECK(check_packed(dev_QW, dev_SW, "QW or SW"));
    if (w_bits == 4 && (uintptr_t)dev_SW % 4) return fail(TAB_ERR_BAD_ARGUMENT, "SW must be aligned to 4 bytes");
    TAB_CHECK(check_rows(dev_Y, dtype, 1, N, N, "Y"));
    const tab::ExpertsPlan plan = tab::experts_plan(dtype, true, w_bits, R, E, N, tab::blocks8(K));
    if (plan.few) {
        const tab::ExpertsArgs a = experts_args(dev_X, nullptr, ldx, M, dev_rows, dev_offsets, dev_QW, dev_SW, w_block_rows, R, E, N, K, dev_Y);
        const hipError_t e = w_bits == 4 ? tab::launch_experts4_few(dtype, plan, a, static_cast<hipStream_t>(stream)) : tab::launch_experts8_few(dtype, plan, a, static_cast<hipStream_t>(stream));
        return e == hipSuccess ? TAB_OK : device_fail(e, "experts launch");
    }
    TAB_CHECK(check_quantize(M, K, 1, false));
    TAB_CHECK(check_workspace(workspace, workspace_bytes, tab_experts_linear_workspace_bytes(dtype, w_bits, M, R, E, N, K)));
    uint8_t *const q = static_cast<uint8_t *>(workspace), *const s = q + packed_numbers(M, K);
    const size_t packed = packed_bytes(M, K);
    TAB_CHECK(tab_quantize8(dev_X, dtype, M, K, ldx, 1, TAB_E4M3, q, s, nullptr, nullptr, stream));
    return tab_experts_linear_packed(q, TAB_E4M3, s, M, dev_rows, dev_offsets, dev_QW, dev_SW, w_bits, w_block_rows, R, E, N, K, dev_Y, dtype, 1, q + packed,
                                     workspace_bytes - packed, stream);
}

int tab_experts_grad_weight(const void *dev_QD, int d_format, const void *dev_SD, const void *dev_QX, const void *dev_SX, const int *dev_offsets, int R, int E, int N,
                            int K, void *dev_dW, int out_dtype, void *stream)
{
    TAB_CHECK(check_format(d_format));
    TAB_CHECK(check_type(out_dtype, "out_dtype"));
    TAB_CHECK(check_runs(R, nullptr, dev_offsets, R, E));
    TAB_CHECK(check_grad_sizes(R, E, N, K, out_dtype));
    TAB_CHECK(check_packed(dev_QD, dev_SD, "QD or SD"));
    TAB_CHECK(check_packed(dev_QX, dev_SX, "QX or SX"));
    TAB_CHECK(check_rows(dev_dW, out_dtype, 1, K, K, "dW"));
    const tab::ExpertsGradArgs a = {static_cast<const uint8_t *>(dev_QD), static_cast<const uint8_t *>(dev_SD), static_cast<const uint8_t *>(dev_QX),
                                    static_cast<const uint8_t *>(dev_SX), dev_dW, dev_offsets, R, E, N, K, tab::run_blocks_most(R, E)};
    const hipError_t e = tab::launch_experts_grad(out_dtype, d_format, a, static_cast<hipStream_t>(stream));
    return e == hipSuccess ? TAB_OK : device_fail(e, "experts gradient launch");
}

int tab_experts_check_gradients(int x_dtype, int w_dtype, int M, int k, int R, int E, int N, int K, int of_x, int of_w)
{
    TAB_CHECK(check_type(x_dtype, "x_dtype"));
    TAB_CHECK(check_type(w_dtype, "w_dtype"));
    if (of_w) {
        TAB_CHECK(check_by_expert_sizes(R, R, E, N));
        TAB_CHECK(check_grad_sizes(R, E, N, K, w_dtype));
    }
    if (of_x) {
        // dY, its rows sorted, times the transposed weights; the rows of a token added up from fp32
        if (!of_w) TAB_CHECK(check_quantize(R, N, 1, false));
        TAB_CHECK(check_experts_sizes(R, false, R, E, K, N, k ? TAB_F32 : x_dtype, x_dtype == TAB_F32, 8));
        if (k) TAB_CHECK(check_combine_sizes(M, k, R, K));
    }
    return TAB_OK;
}

static int check_combine(int M, int k, int R, int D, const int *places, const float *weights)
{
    TAB_CHECK(check_combine_sizes(M, k, R, D));
    TAB_CHECK(check_int32(places, "places"));
    return check_int32(weights, "weights", true);
}

int tab_combine(const void *dev_Y, int dtype, const int *dev_places, const float *dev_weights, int M, int k, int R, int D, void *dev_out, int out_dtype, void *stream)
{
    TAB_CHECK(check_type(dtype, "dtype"));
    TAB_CHECK(check_type(out_dtype, "out_dtype"));
    if (dtype != out_dtype && dtype != TAB_F32) return fail(TAB_ERR_BAD_ARGUMENT, "out_dtype must be dtype, or dtype 0 (fp32)");
    TAB_CHECK(check_combine(M, k, R, D, dev_places, dev_weights));
    TAB_CHECK(check_rows(dev_Y, dtype, 1, D, D, "Y"));
    TAB_CHECK(check_rows(dev_out, out_dtype, 1, D, D, "out"));
    const tab::CombineArgs a = {dev_Y, dev_places, dev_weights, dev_out, M, k, R, D};
    const hipError_t e = tab::launch_combine(dtype, out_dtype, a, static_cast<hipStream_t>(stream));
    return e == hipSuccess ? TAB_OK : device_fail(e, "combine launch");
}

int tab_combine_backward(const void *dev_dout, const void *dev_Y, int dtype, const int *dev_places, const float *dev_weights, const int *dev_used, int M, int k, int R,
                         int D, void *dev_dY, float *dev_dweights, void *stream)
{
    TAB_CHECK(check_type(dtype, "dtype"));
    TAB_CHECK(check_combine(M, k, R, D, dev_places, dev_weights));
    TAB_CHECK(check_int32(dev_used, "used", true));
    TAB_CHECK(check_rows(dev_dout, dtype, 1, D, D, "dout"));
    if (!dev_dY && !dev_dweights) return fail(TAB_ERR_BAD_ARGUMENT, "null device pointer: dY and dweights");
    if (dev_dY) TAB_CHECK(check_rows(dev_dY, dtype, 1, D, D, "dY"));
    if (dev_dweights) {
        TAB_CHECK(check_rows(dev_Y, dtype, 1, D, D, "Y"));
        TAB_CHECK(check_int32(dev_dweights, "dweights"));
    }
    const tab::CombineGradArgs a = {dev_dout, dev_Y, dev_places, dev_used, dev_weights, dev_dY, dev_dweights, M, k, R, D};
    const hipError_t e = tab::launch_combine_grad(dtype, a, static_cast<hipStream_t>(stream));
    return e == hipSuccess ? TAB_OK : device_fail(e, "combine gradient launch");
}

/* Test hook, absent from include/tab_amd.h: how a product over experts would be computed: 0 as few rows, else (the tile's rows + columns) / 2 * 100 + the
 * parts of K. */
int tab_internal_experts_way(int out_dtype, int w_bits, int R, int E, int N, int K)
{
    const tab::ExpertsPlan plan = tab::experts_plan(out_dtype, true, w_bits, R, E, N, tab::blocks8(K));
    return plan.few ? 0 : (plan.rows + plan.columns) / 2 * 100 + plan.parts;
}

/* The same of the gradients of the weights: the tile. */
int tab_internal_experts_grad_way(int out_dtype, int R, int E, int N, int K) { return tab::experts_grad_way(out_dtype, R, E, N, K); }

}  // extern "C"
