// Launches of the products over experts for one kind of weight (WBITS 8 or 4): the kernels are those of one weight (tab_linear8_tiles.h), with rows by
// expert.
#pragma once
#include "tab_linear8_tiles.h"

namespace tab {

namespace {

template <int FORMAT, int OUT, bool EXACT, int WBITS>
hipError_t launch_expert_tiles(const ExpertsPlan &plan, const ExpertTileParams &p, hipStream_t stream)
{
    return launch_tiles<FORMAT, OUT, EXACT, WBITS, kRowsByExpert>(Plan8{plan.rows, plan.columns, plan.parts, plan.kb_per_part, 0}, plan.workgroups, p, stream);
}

template <int FORMAT, int WBITS>
hipError_t launch_expert_product(int out, bool full_sums, const ExpertsPlan &plan, const ExpertsArgs &a, int scale_rows, void *workspace, hipStream_t stream)
{
    ExpertTileParams p = {};
    static_cast<TileParams &>(p) = TileParams{static_cast<const uint8_t *>(a.x), a.sx, a.qw, a.sw, plan.parts > 1 ? workspace : a.y, a.R, a.N, a.KB, scale_rows, plan.kb_per_part,
                                              (int)run_tiles_most(a.R, a.E, plan.rows), (a.N + plan.columns - 1) / plan.columns};
    p.offsets = a.offsets, p.rows = a.rows, p.E = a.E, p.x_rows = a.x_rows;
    if (plan.parts == 1 && out != 0)
        return out == 1 ? launch_expert_tiles<FORMAT, 1, false, WBITS>(plan, p, stream) : launch_expert_tiles<FORMAT, 2, false, WBITS>(plan, p, stream);
    const hipError_t e = out == 0 && full_sums ? launch_expert_tiles<FORMAT, 0, true, WBITS>(plan, p, stream) : launch_expert_tiles<FORMAT, 0, false, WBITS>(plan, p, stream);
    return e != hipSuccess || plan.parts == 1 ? e : launch_join(out, static_cast<const float *>(workspace), a.y, (long)a.R * a.N, plan.parts, stream);
}

template <int INPUT, int FORMAT, int OUT, int WBITS> hipError_t launch_expert_rows(const ExpertsPlan &plan, const ExpertsArgs &a, int scale_rows, hipStream_t stream)
{
    ExpertRowsParams p = {};
    static_cast<RowsParams &>(p) = RowsParams{a.x, a.sx, a.qw, a.sw, a.y, a.R, a.N, a.K, a.KB, scale_rows, plan.columns, a.ldx, make_div32((uint32_t)a.KB)};
    p.offsets = a.offsets, p.rows = a.rows, p.E = a.E, p.x_rows = a.x_rows, p.each = plan.parts, p.most = plan.most;
    const unsigned n = (unsigned)plan.workgroups, lds = (unsigned)rows_lds(plan.most, a.KB);
    if (plan.most <= 16) linear8_rows<INPUT, FORMAT, OUT, 1, WBITS, kRowsByExpert><<<n, 64 * kRowsWaves, lds, stream>>>(p);
    else linear8_rows<INPUT, FORMAT, OUT, 2, WBITS, kRowsByExpert><<<n, 64 * kRowsWaves, lds, stream>>>(p);
    return hipGetLastError();
}

template <int WBITS> hipError_t launch_expert_few(int dtype, const ExpertsPlan &plan, const ExpertsArgs &a, int scale_rows, hipStream_t stream)
{
    return dtype == 0 ? launch_expert_rows<0, 0, 0, WBITS>(plan, a, scale_rows, stream)
                      : dtype == 1 ? launch_expert_rows<1, 0, 1, WBITS>(plan, a, scale_rows, stream) : launch_expert_rows<2, 0, 2, WBITS>(plan, a, scale_rows, stream);
}

}  // namespace

}  // namespace tab
