// Products of rows sorted by expert with 8-bit weights, and the rule that picks their kernel.
#include "tab_experts_launch.h"

namespace tab {

// Few rows to an expert: the launch whose workgroups hold an expert's rows in LDS and stream its weight; `columns` is then the groups of 16 rows of a weight
// that a workgroup takes, `parts` the workgroups to an expert.
ExpertsPlan experts_plan(int out, int R, int E, int N, int KB)
{
    ExpertsPlan plan = {};
    const int active = E < R ? E : R;
    if ((long)R <= 8L * active && rows_fit(1, KB)) {
        int most = R < 16 ? R : 16;
        while (!rows_fit(most, KB)) most--;
        const int groups = (N + 15) / 16;
        const long experts = E + 1L < R ? E + 1L : R;
        const long each = (groups * experts + 1023) / 1024;
        plan = {true, most, 0, (int)each, (int)((groups + each - 1) / each), 0, 0};
        plan.workgroups = experts * plan.parts;
        return plan;
    }
    // as plan8, by the tiles that `active` experts of like numbers of rows come to
    constexpr TileTimes kFast[] = {{64, 64, 3, 0.05, 0.174, 0.8}, {64, 128, 2, 0.171, 0.242, 1.37}, {128, 128, 2, 0.571, 0.473, 1.69}, {256, 256, 1, 1.235, 1.125, 6.25}};
    constexpr TileTimes kExact[] = {{64, 64, 3, 0.371, 0.242, 0.7}, {64, 128, 2, 0.553, 0.336, 1.32}, {128, 128, 2, 1.22, 0.716, 1.65}};
    const double join = out == 0 ? 2.5 : 1.9, join_part = out == 0 ? 0.936e-6 : 0.747e-6, join_out = out == 0 ? 0.008e-6 : 0;
    double least = 1e30;
    for (int i = 0; i < (out == 0 ? 3 : 4); i++) {
        const TileTimes &tile = out == 0 ? kExact[i] : kFast[i];
        const long columns = ((long)N + tile.columns - 1) / tile.columns, most = run_tiles_most(R, E, tile.rows) * columns;
        const double rows = R <= (long)active * tile.rows / 2 ? active : (double)R / tile.rows + 0.5 * active;
        for (int parts = 1; parts <= 16 && parts <= KB; parts *= 2) {
            if (parts > 1 && rows * (double)columns * parts > 2048) break;
            const int steps = (KB + parts - 1) / parts;
            if ((KB + steps - 1) / steps != parts) continue;
            const double each = __builtin_ceil(rows * (double)columns * parts / 256), rounds = __builtin_ceil(each / tile.held);
            const double alone = tile.alone * rounds, among = tile.among * each;
            double t = steps * (alone > among ? alone : among) + tile.out * each * (parts > 1 || out == 0 ? 2 : 1);
            if (parts > 1) t += join + (parts * join_part + join_out) * (double)R * (double)N;
            if (t < least) {
                least = t;
                plan = {false, 0, tile.rows, tile.columns, parts, steps, most * parts};
            }
        }
    }
    return plan;
}

hipError_t launch_experts8(int out, bool full_sums, int x_format, const ExpertsPlan &plan, const ExpertsArgs &a, void *workspace, hipStream_t stream)
{
    const int scale_rows = w_scale_rows(a.N, a.w_block_rows);
    if (plan.few) {
        if (x_format == 0)
            return out == 0 ? launch_expert_rows<3, 0, 0, 8>(plan, a, scale_rows, stream)
                            : out == 1 ? launch_expert_rows<3, 0, 1, 8>(plan, a, scale_rows, stream) : launch_expert_rows<3, 0, 2, 8>(plan, a, scale_rows, stream);
        return out == 0 ? launch_expert_rows<3, 1, 0, 8>(plan, a, scale_rows, stream)
                        : out == 1 ? launch_expert_rows<3, 1, 1, 8>(plan, a, scale_rows, stream) : launch_expert_rows<3, 1, 2, 8>(plan, a, scale_rows, stream);
    }
    return x_format == 0 ? launch_expert_product<0, 8>(out, full_sums, plan, a, scale_rows, workspace, stream)
                         : launch_expert_product<1, 8>(out, full_sums, plan, a, scale_rows, workspace, stream);
}

hipError_t launch_experts8_few(int dtype, const ExpertsPlan &plan, const ExpertsArgs &a, hipStream_t stream)
{
    return launch_expert_few<8>(dtype, plan, a, w_scale_rows(a.N, a.w_block_rows), stream);
}

}  // namespace tab
