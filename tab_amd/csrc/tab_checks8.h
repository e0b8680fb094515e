// Argument checks that the C ABI's files of the 8-bit and 4-bit layers, the norms and the experts share.
#pragma once
#include "../../include/tab_amd.h"
#include "tab_blocks8.h"

using tab::device_fail;
using tab::fail;

namespace {  // one copy a file

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
