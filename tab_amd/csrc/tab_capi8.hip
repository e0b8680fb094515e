// C ABI of the 8-bit layers and of the norms around a block: argument checks and launches.  No allocation, no synchronisation, no
// host<->device copy.
#include "../../include/tab_amd.h"
#include "tab_blocks8.h"

using tab::device_fail;
using tab::fail;

namespace {

constexpr long kMostThreads = 0xffffffffL;  // of one launch
constexpr int kMostRows = 0x7fffffff - 512;

int element_bytes(int dtype) { return dtype == TAB_F32 ? 4 : 2; }

int check_type(int dtype, const char *what)
{
    return dtype >= TAB_F32 && dtype <= TAB_F16 ? TAB_OK : fail(TAB_ERR_BAD_ARGUMENT, "%s must be 0 (fp32), 1 (bf16) or 2 (fp16), got %d", what, dtype);
}

int check_format(int format)
{
    return format == TAB_E4M3 || format == TAB_E5M2 ? TAB_OK : fail(TAB_ERR_BAD_ARGUMENT, "format must be 0 (E4M3) or 1 (E5M2), got %d", format);
}

int check_block_rows(int rows)
{
    return rows == 1 || rows == tab::kBlock8 ? TAB_OK : fail(TAB_ERR_BAD_ARGUMENT, "blocks must have 1 or 128 rows, got %d", rows);
}

// A matrix of `rows` rows, `ld` elements apart
int check_rows(const void *p, int dtype, int rows, int columns, long ld, const char *what)
{
    if (!p) return fail(TAB_ERR_BAD_ARGUMENT, "null device pointer: %s", what);
    if ((uintptr_t)p % element_bytes(dtype)) return fail(TAB_ERR_BAD_ARGUMENT, "%s must be aligned to its elements", what);
    if (rows > 1 && (ld < columns || ld > 0x7fffffffL))
        return fail(TAB_ERR_BAD_ARGUMENT, "row stride of %s must be at least %d and below 2^31, got %ld", what, columns, ld);
    return TAB_OK;
}

int check_packed(const void *q, const void *s, const char *what)
{
    if (!q || !s) return fail(TAB_ERR_BAD_ARGUMENT, "null device pointer: %s", what);
    if ((uintptr_t)q % 16) return fail(TAB_ERR_BAD_ARGUMENT, "%s must be aligned to 16 bytes", what);
    return TAB_OK;
}

int check_workspace(const void *workspace, size_t bytes, size_t need)
{
    if (need && (!workspace || bytes < need || (uintptr_t)workspace % 16))
        return fail(TAB_ERR_WORKSPACE, "workspace must hold %zu bytes, 16-byte aligned (got %zu)", need, bytes);
    return TAB_OK;
}

int check_linear(int out_dtype, int M, int N, int K)
{
    if (M < 1 || N < 1 || K < 1) return fail(TAB_ERR_BAD_ARGUMENT, "M, N, K must be positive");
    if (M > kMostRows || N > kMostRows || tab::blocks8(K) > tab::kBlocks8Most) return fail(TAB_ERR_BAD_SHAPE, "product too large for 32-bit offsets into a tile");
    if (tab::linear8_threads(out_dtype, M, N, tab::blocks8(K)) > kMostThreads) return fail(TAB_ERR_BAD_SHAPE, "product too large for one launch");
    return TAB_OK;
}

int check_quantize(int M, int K, int block_rows, bool transposed)
{
    if (M < 1 || K < 1) return fail(TAB_ERR_BAD_ARGUMENT, "M and K must be positive");
    if (M > kMostRows || tab::quantize8_tiles(block_rows, transposed, M, K) * 256 > kMostThreads) return fail(TAB_ERR_BAD_SHAPE, "matrix too large for one launch");
    return TAB_OK;
}

// the packed activation of tab_linear8 in its workspace: numbers, then scales
size_t align16(size_t n) { return (n + 15) / 16 * 16; }
size_t packed_numbers(int M, int K) { return (size_t)M * tab::blocks8(K) * tab::kBlock8; }
size_t packed_bytes(int M, int K) { return packed_numbers(M, K) + align16((size_t)M * tab::blocks8(K)); }

#define TAB_CHECK(call)                              \
    do {                                             \
        const int status_of_check = (call);          \
        if (status_of_check != TAB_OK) return status_of_check; \
    } while (0)

}  // namespace

extern "C" {

int tab_blocks8(int K) { return K < 1 ? 0 : tab::blocks8(K); }

int tab_quantize8(const void *dev_X, int dtype, int M, int K, long ldx, int block_rows, int format, void *dev_Q, void *dev_S, void *dev_QT,
                  void *dev_ST, void *stream)
{
    TAB_CHECK(check_type(dtype, "dtype"));
    TAB_CHECK(check_format(format));
    TAB_CHECK(check_block_rows(block_rows));
    TAB_CHECK(check_quantize(M, K, block_rows, dev_QT != nullptr));
    TAB_CHECK(check_rows(dev_X, dtype, M, K, ldx, "X"));
    if (!dev_Q && !dev_QT) return fail(TAB_ERR_BAD_ARGUMENT, "null device pointer: Q and QT");
    if (dev_Q || dev_S) TAB_CHECK(check_packed(dev_Q, dev_S, "Q or S"));
    if (dev_QT || dev_ST) TAB_CHECK(check_packed(dev_QT, dev_ST, "QT or ST"));
    const tab::Quantize8Args a = {dev_X, static_cast<uint8_t *>(dev_Q), static_cast<uint8_t *>(dev_S), static_cast<uint8_t *>(dev_QT),
                                  static_cast<uint8_t *>(dev_ST), M, K, ldx};
    const hipError_t e = tab::launch_quantize8(dtype, format, block_rows, a, static_cast<hipStream_t>(stream));
    return e == hipSuccess ? TAB_OK : device_fail(e, "quantize8 launch");
}

size_t tab_linear8_packed_workspace_bytes(int out_dtype, int M, int N, int K)
{
    return M < 1 || N < 1 || K < 1 ? 0 : tab::linear8_workspace(out_dtype, M, N, tab::blocks8(K));
}

int tab_linear8_packed(const void *dev_QX, int x_format, const void *dev_SX, const void *dev_QW, const void *dev_SW, int w_block_rows, int M, int N,
                       int K, void *dev_Y, int out_dtype, void *workspace, size_t workspace_bytes, void *stream)
{
    TAB_CHECK(check_format(x_format));
    TAB_CHECK(check_type(out_dtype, "out_dtype"));
    TAB_CHECK(check_block_rows(w_block_rows));
    TAB_CHECK(check_linear(out_dtype, M, N, K));
    TAB_CHECK(check_packed(dev_QX, dev_SX, "QX or SX"));
    TAB_CHECK(check_packed(dev_QW, dev_SW, "QW or SW"));
    TAB_CHECK(check_rows(dev_Y, out_dtype, 1, N, N, "Y"));
    TAB_CHECK(check_workspace(workspace, workspace_bytes, tab_linear8_packed_workspace_bytes(out_dtype, M, N, K)));
    const tab::Linear8Args a = {static_cast<const uint8_t *>(dev_QX), static_cast<const uint8_t *>(dev_SX), static_cast<const uint8_t *>(dev_QW),
                                static_cast<const uint8_t *>(dev_SW), dev_Y, M, N, tab::blocks8(K), w_block_rows};
    const hipError_t e = tab::launch_linear8(out_dtype, x_format, a, workspace, static_cast<hipStream_t>(stream));
    return e == hipSuccess ? TAB_OK : device_fail(e, "linear8 launch");
}

size_t tab_linear8_workspace_bytes(int dtype, int M, int N, int K)
{
    if (M < 1 || N < 1 || K < 1 || tab::linear8_rows_supported(M, K)) return 0;
    return packed_bytes(M, K) + tab_linear8_packed_workspace_bytes(dtype, M, N, K);
}

int tab_linear8(const void *dev_X, int dtype, long ldx, const void *dev_QW, const void *dev_SW, int w_block_rows, int M, int N, int K, void *dev_Y,
                void *workspace, size_t workspace_bytes, void *stream)
{
    TAB_CHECK(check_type(dtype, "dtype"));
    TAB_CHECK(check_block_rows(w_block_rows));
    TAB_CHECK(check_linear(dtype, M, N, K));
    TAB_CHECK(check_rows(dev_X, dtype, M, K, ldx, "X"));
    TAB_CHECK(check_packed(dev_QW, dev_SW, "QW or SW"));
    TAB_CHECK(check_rows(dev_Y, dtype, 1, N, N, "Y"));
    if (tab::linear8_rows_supported(M, K)) {
        const tab::Linear8RowsArgs a = {dev_X, static_cast<const uint8_t *>(dev_QW), static_cast<const uint8_t *>(dev_SW), dev_Y, M, N, K, w_block_rows, ldx};
        const hipError_t e = tab::launch_linear8_rows(dtype, a, static_cast<hipStream_t>(stream));
        return e == hipSuccess ? TAB_OK : device_fail(e, "linear8 launch");
    }
    TAB_CHECK(check_quantize(M, K, 1, false));
    TAB_CHECK(check_workspace(workspace, workspace_bytes, tab_linear8_workspace_bytes(dtype, M, N, K)));
    uint8_t *const q = static_cast<uint8_t *>(workspace), *const s = q + packed_numbers(M, K);
    const size_t packed = packed_bytes(M, K);
    TAB_CHECK(tab_quantize8(dev_X, dtype, M, K, ldx, 1, TAB_E4M3, q, s, nullptr, nullptr, stream));
    return tab_linear8_packed(q, TAB_E4M3, s, dev_QW, dev_SW, w_block_rows, M, N, K, dev_Y, dtype, q + packed, workspace_bytes - packed, stream);
}

// What both directions of the norms share: sizes, types and the gate.
static int check_norm(int dtype, int M, int D, const void *block, const void *gate, int gate_dtype, int gates, const float *w_post, const float *w_pre,
                      float alpha, float eps)
{
    TAB_CHECK(check_type(dtype, "dtype"));
    if (M < 1 || D < 1) return fail(TAB_ERR_BAD_ARGUMENT, "M and D must be positive");
    if (M > kMostRows || D > tab::kNormWidthMost) return fail(TAB_ERR_BAD_SHAPE, "rows may have at most %d elements, got %d", tab::kNormWidthMost, D);
    if (!(eps >= 0.f)) return fail(TAB_ERR_BAD_ARGUMENT, "eps must not be negative");
    if (!block && (gate || w_post || alpha != 1.f)) return fail(TAB_ERR_BAD_ARGUMENT, "a gate, w_post and alpha belong to a block's output Y");
    if (gate) {
        if (gate_dtype != TAB_F32 && gate_dtype != dtype) return fail(TAB_ERR_BAD_ARGUMENT, "gate_dtype must be 0 (fp32) or dtype, got %d", gate_dtype);
        if (gates < 1 || M % gates) return fail(TAB_ERR_BAD_ARGUMENT, "M must be a multiple of gates, got %d and %d", M, gates);
        TAB_CHECK(check_rows(gate, gate_dtype, gates, D, D, "gate"));
    }
    if (((uintptr_t)w_post | (uintptr_t)w_pre) % 4) return fail(TAB_ERR_BAD_ARGUMENT, "w_post and w_pre must be aligned to their elements");
    return TAB_OK;
}

int tab_norm_residual(const void *dev_X, long ldx, const void *dev_Y, long ldy, const void *dev_gate, int gate_dtype, int gates,
                      const float *dev_w_post, const float *dev_w_pre, float alpha, float eps, int dtype, int M, int D, void *dev_R, void *dev_H,
                      void *dev_S, void *stream)
{
    TAB_CHECK(check_norm(dtype, M, D, dev_Y, dev_gate, gate_dtype, gates, dev_w_post, dev_w_pre, alpha, eps));
    TAB_CHECK(check_rows(dev_X, dtype, M, D, ldx, "X"));
    if (dev_Y) {
        TAB_CHECK(check_rows(dev_Y, dtype, M, D, ldy, "Y"));
        TAB_CHECK(check_rows(dev_R, dtype, 1, D, D, "R"));
    } else if (dev_R) {
        return fail(TAB_ERR_BAD_ARGUMENT, "R is X where there is no Y");
    }
    if (dev_S) TAB_CHECK(check_packed(dev_H, dev_S, "H or S"));
    else if (dev_H) TAB_CHECK(check_rows(dev_H, dtype, 1, D, D, "H"));
    else if (!dev_Y) return fail(TAB_ERR_BAD_ARGUMENT, "null device pointer: H");
    const tab::NormArgs a = {dev_X, dev_Y, dev_gate, dev_w_post, dev_w_pre, dev_R, dev_H, static_cast<uint8_t *>(dev_S), M, D,
                             dev_gate ? M / gates : M, ldx, ldy, alpha, eps};
    const hipError_t e = tab::launch_norm(dtype, gate_dtype, a, static_cast<hipStream_t>(stream));
    return e == hipSuccess ? TAB_OK : device_fail(e, "norm launch");
}

size_t tab_norm_residual_backward_workspace_bytes(int M, int D, int gates)
{
    if (M < 1 || D < 1 || D > tab::kNormWidthMost || gates < 0 || (gates > 0 && M % gates)) return 0;
    return tab::norm_grad_workspace(gates != 0, M, D, gates ? M / gates : M);
}

int tab_norm_residual_backward(const void *dev_dR, const void *dev_dH, const void *dev_R, const void *dev_Y, const void *dev_gate, int gate_dtype,
                               int gates, const float *dev_w_post, const float *dev_w_pre, float alpha, float eps, int dtype, int M, int D,
                               void *dev_dX, void *dev_dY, void *dev_dgate, float *dev_dw_post, float *dev_dw_pre, void *workspace,
                               size_t workspace_bytes, void *stream)
{
    TAB_CHECK(check_norm(dtype, M, D, dev_Y, dev_gate, gate_dtype, gates, dev_w_post, dev_w_pre, alpha, eps));
    if (!dev_dR && !dev_dH) return fail(TAB_ERR_BAD_ARGUMENT, "null device pointer: dR and dH");
    if (dev_dR) TAB_CHECK(check_rows(dev_dR, dtype, 1, D, D, "dR"));
    if (dev_dH) {
        TAB_CHECK(check_rows(dev_dH, dtype, 1, D, D, "dH"));
        TAB_CHECK(check_rows(dev_R, dtype, 1, D, D, "R"));
    }
    TAB_CHECK(check_rows(dev_dX, dtype, 1, D, D, "dX"));
    if (dev_Y) {
        TAB_CHECK(check_rows(dev_Y, dtype, 1, D, D, "Y"));
        TAB_CHECK(check_rows(dev_dY, dtype, 1, D, D, "dY"));
    }
    if ((dev_dgate && !dev_gate) || (!dev_Y && (dev_dY || dev_dw_post)))
        return fail(TAB_ERR_BAD_ARGUMENT, "gradients of operands that are not there");
    if (dev_dgate) TAB_CHECK(check_rows(dev_dgate, gate_dtype, 1, D, D, "dgate"));
    if (((uintptr_t)dev_dw_post | (uintptr_t)dev_dw_pre) % 4) return fail(TAB_ERR_BAD_ARGUMENT, "dw_post and dw_pre must be aligned to their elements");
    TAB_CHECK(check_workspace(workspace, workspace_bytes, tab_norm_residual_backward_workspace_bytes(M, D, dev_gate ? gates : 0)));
    const tab::NormGradArgs a = {dev_dR, dev_dH, dev_R, dev_Y, dev_gate, dev_w_post, dev_w_pre, dev_dX, dev_dY, dev_dgate, dev_dw_post, dev_dw_pre,
                                 M, D, dev_gate ? M / gates : M, alpha, eps};
    const hipError_t e = tab::launch_norm_grad(dtype, gate_dtype, a, static_cast<float *>(workspace), static_cast<hipStream_t>(stream));
    return e == hipSuccess ? TAB_OK : device_fail(e, "norm gradient launch");
}

/* Test hook, absent from include/tab_amd.h: how an M x N product over K would be computed: 0 as few rows, else (the tile's rows + columns) / 2 * 100
 * + the parts of K. */
int tab_internal_linear8_way(int out_dtype, int M, int N, int K) { return tab::linear8_way(out_dtype, M, N, tab::blocks8(K)); }

}  // extern "C"
