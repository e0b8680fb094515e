// Products of rows sorted by expert with 8-bit weights, and the rule that picks their kernel.  16384 rows, bf16: 32 experts of 2048 x 4096 150-159 us, 1.75-1.8 PFLOP/s
// (640 tiles of 256 x 256 with a quarter of their rows empty, 2.5 rounds of the chip; 512 rows each 124, one weight for all 107, as linear8's kernel); 16 of 2048 x 2048
// 82-90 (1024 rows each 64), rows in fp32 100-104.
#include "tab_experts_launch.h"

namespace tab {

namespace {

// The experts that R rows come to, where each takes any
double chosen_experts(int R, int E) { return E > 1 ? E * (1 - __builtin_pow(1 - 1.0 / E, R)) : 1; }

}  // namespace

// The least of what the ways take, us: few rows to an expert in one launch (waves stream KB of the weights, workgroups take turns on the CUs), or the launches of
// the quantizer and of tiles (as plan8 has them, by the tiles that the chosen experts come to).  Constants fitted to every way of 460 products of 1 .. 20000
// rows over 1 .. 137 experts of 64 .. 5000 columns and K, 8 and 4 bits, on an MI355X; what the rule picks takes 3 % longer than the best of them in the
// mean, 1.65 times at most (15 rows of 31 experts of 2048 x 3456).
ExpertsPlan experts_plan(int out, bool full_sums, int bits, int R, int E, int N, int KB)
{
    const bool exact = out == 0 && full_sums;
    const double chosen = chosen_experts(R, E), weight_mb = chosen * N * (double)KB * (kBlock8 * bits / 8 * 1e-6);
    ExpertsPlan plan = {};
    double least = 1e30;
    if ((long)R <= 40L * (E < R ? E : R) && rows_fit(1, KB)) {
        int most = 16;
        while (!rows_fit(most, KB)) most /= 2;
        const double crowd = (double)R / E - 2.6, runs = chosen * (crowd > 0 ? 1 + crowd / most : 1);
        for (int split = 1; split <= kRowsWaves && split <= KB; split *= 2) {
            const long groups = (N + 15) / 16;
            const double wave_kb = 16e-3 * KB * kBlock8 * bits / 8 / split, workgroups = runs * (double)((groups * split + kRowsWaves - 1) / kRowsWaves);
            const double all = wave_kb / 4.46 + workgroups / 256 * (1.44 + wave_kb / 4.09), t = 4.24 + (weight_mb / 5.94 > all ? weight_mb / 5.94 : all);
            if (t < least) {
                least = t;
                const int columns = kRowsWaves / split * 16;
                plan = {true, most, columns, split, 0, run_tiles_most(R, E, most) * ((N + columns - 1L) / columns)};
            }
        }
    }
    const double join = out == 0 ? 2.5 : 1.9, join_part = out == 0 ? 0.936e-6 : 0.747e-6, mb = weight_mb + R * (double)N * (out == 0 ? 4e-6 : 2e-6);
    for (int i = 0; i < (exact ? 3 : 4); i++) {
        const TileTimes &tile = exact ? kExpertExact[i] : kExpertTiles[i];
        const long columns = ((long)N + tile.columns - 1) / tile.columns, most = run_tiles_most(R, E, tile.rows) * columns;
        const double spread = (double)R / tile.rows + 0.79 * chosen, rows = spread > chosen ? spread : chosen;
        for (int parts = 1; parts <= 16 && parts <= KB; parts *= 2) {
            if (parts > 1 && rows * (double)columns * parts > 2048) break;
            const int steps = (KB + parts - 1) / parts;
            if ((KB + steps - 1) / steps != parts) continue;
            const double each = __builtin_ceil(rows * (double)columns * parts / 256), rounds = __builtin_ceil(each / tile.held);
            const double alone = tile.alone * rounds, among = tile.among * each;
            double t = steps * (alone > among ? alone : among) + tile.out * each * (parts > 1 || out == 0 ? 2 : 1);
            if (parts > 1) t += join + parts * join_part * (double)R * (double)N;
            t = 7 + (t > mb / 5.73 ? t : mb / 5.73);
            if (t < least) {
                least = t;
                plan = {false, tile.rows, tile.columns, parts, steps, most * parts};
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
