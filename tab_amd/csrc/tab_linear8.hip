// Launches of the product of packed 8-bit operands (tab_linear8_tiles.h).
#include "tab_linear8_tiles.h"

namespace tab {

size_t linear8_workspace(int out_dtype, int M, int N, int KB)
{
    if (rows_fit(M, KB)) return 0;
    const Plan8 plan = plan8(out_dtype, M, N, KB);
    return plan.parts > 1 ? (size_t)plan.parts * (size_t)M * (size_t)N * sizeof(float) : 0;
}

long linear8_threads(int out_dtype, int M, int N, int KB)
{
    if (rows_fit(M, KB)) return 0;  // (at most 512 workgroups)
    const Plan8 plan = plan8(out_dtype, M, N, KB);
    return plan.tiles * plan.parts * threads_of(plan);
}

int linear8_way(int out_dtype, int M, int N, int KB)
{
    if (rows_fit(M, KB)) return 0;
    const Plan8 plan = plan8(out_dtype, M, N, KB);
    return (plan.rows + plan.columns) / 2 * 100 + plan.parts;
}

hipError_t launch_linear8(int out_dtype, int x_format, const Linear8Args &a, void *workspace, hipStream_t stream)
{
    const int scale_rows = w_scale_rows(a.N, a.w_block_rows);
    return x_format == 0 ? launch_product<0, 8>(out_dtype, a, scale_rows, workspace, stream) : launch_product<1, 8>(out_dtype, a, scale_rows, workspace, stream);
}

bool linear8_rows_supported(int M, int K) { return rows_fit(M, blocks8(K)); }

hipError_t launch_linear8_rows(int dtype, const Linear8RowsArgs &a, hipStream_t stream)
{
    const RowsParams p = {a.x, nullptr, a.qw, a.sw, a.y, a.M, a.N, a.K, blocks8(a.K), w_scale_rows(a.N, a.w_block_rows), 0, 0, a.ldx, make_div32((uint32_t)blocks8(a.K))};
    return dtype == 0 ? launch_rows<0, 0, 0>(p, stream) : dtype == 1 ? launch_rows<1, 0, 1>(p, stream) : launch_rows<2, 0, 2>(p, stream);
}

}  // namespace tab
