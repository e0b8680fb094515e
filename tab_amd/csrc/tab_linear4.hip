// Product of a packed 8-bit activation and weights of 4 bits (E2M1) with a power-of-two scale per group of 32,
//   Y[m][n] = sum over kb of 2^(SX[kb][m] - 127) * sum over groups g of 2^(SW[kb][n][g] - 127) * sum over k in g of QX[m][k] QW[n][k].
//
// The kernels are those of the 8-bit product (tab_linear8_tiles.h): the matrix instruction takes E4M3 and E2M1 side by side, at the rate of its wider operand,
// and a scale for each lane's 32 numbers, so a group's scale costs a shift a row of W and step.  What changes is W's way: half the bytes from memory and
// into LDS, which is all that few rows are bound by.  4096 x 4096 x 4096, bf16: 57 us with X's quantizer (9.6) and a launch, the product 49.6 (2.77 PFLOP/s, what the
// 8-bit product reaches at 8192^3); one row of 4096: 4.2 us, 8.9 MB, of which a launch is 2.5.
#include "tab_linear8_tiles.h"

namespace tab {

bool linear4_rows_supported(int M, int N, int K) { return rows_way<4>(M, N, blocks8(K)); }

size_t linear4_workspace(int out_dtype, int M, int N, int KB)
{
    if (rows_way<4>(M, N, KB)) return 0;
    const Plan8 plan = plan8(out_dtype, M, N, KB);
    return plan.parts > 1 ? (size_t)plan.parts * (size_t)M * (size_t)N * sizeof(float) : 0;
}

hipError_t launch_linear4(int out_dtype, const Linear8Args &a, void *workspace, hipStream_t stream) { return launch_product<0, 4>(out_dtype, a, a.N, workspace, stream); }

hipError_t launch_linear4_rows(int dtype, const Linear8RowsArgs &a, hipStream_t stream)
{
    const RowsParams p = {a.x, nullptr, a.qw, a.sw, a.y, a.M, a.N, a.K, blocks8(a.K), a.N, 0, 0, a.ldx, make_div32((uint32_t)blocks8(a.K))};
    return dtype == 0 ? launch_rows<0, 0, 0, 4>(p, stream) : dtype == 1 ? launch_rows<1, 0, 1, 4>(p, stream) : launch_rows<2, 0, 2, 4>(p, stream);
}

}  // namespace tab
