// Gradients of the experts' weights: dW[e] = sum over the rows r of expert e of dY[r]^T X[r], from both operands packed along the rows by blocks of 128 that
// belong to one expert.  Every expert has the same tiles, and a tile goes through its expert's own blocks.  16384 rows, 16 experts of 2048 x 2048, E5M2: 97-100 us, 1.4
// PFLOP/s: 1024 tiles of 256 x 256, four rounds of the chip with some eight steps each, so the way in and out of a tile takes more than half of its time.
#include "tab_linear8_tiles.h"

namespace tab {

namespace {

// As plan8, where every expert has the same tiles, with some half a block more than its share of the rows; `start` us of a round of the chip.  Fitted to every tile of
// 60 gradients (1 .. 90 experts, 20 .. 16000 rows); what the rule picks takes 3 % longer than the best of them in the mean, 1.45 times at most (65 experts of
// 237 x 247).
Plan8 grad_plan(int out, int R, int E, int M, int N)
{
    constexpr double kOut[] = {0.64, 1.43, 2.04, 3.02}, kStart[] = {0.87, 0.43, 0.83, 5.95};
    const double chosen = E > 1 ? E * (1 - __builtin_pow(1 - 1.0 / E, R)) : 1, steps = R / chosen / kBlock8 + 0.5;
    Plan8 best = {};
    double least = 1e30;
    for (int i = 0; i < (out == 0 ? 3 : 4); i++) {
        const TileTimes &tile = out == 0 ? kExpertExact[i] : kExpertTiles[i];
        const long tiles = ((M + (long)tile.rows - 1) / tile.rows) * ((N + (long)tile.columns - 1) / tile.columns);
        const double each = __builtin_ceil((double)tiles * E / 256), rounds = __builtin_ceil(each / tile.held);
        const double alone = tile.alone * rounds, among = tile.among * each;
        const double t = steps * (alone > among ? alone : among) + kOut[i] * each * (out == 0 ? 2 : 1) + kStart[i] * rounds;
        if (t < least) {
            least = t;
            best = {tile.rows, tile.columns, 1, 0, tiles};
        }
    }
    return best;
}

template <int FORMAT> hipError_t launch(int out, const Plan8 &plan, long workgroups, const ExpertTileParams &p, hipStream_t stream)
{
    return out == 0 ? launch_tiles<FORMAT, 0, true, 8, kKByExpert>(plan, workgroups, p, stream)
                    : out == 1 ? launch_tiles<FORMAT, 1, false, 8, kKByExpert>(plan, workgroups, p, stream) : launch_tiles<FORMAT, 2, false, 8, kKByExpert>(plan, workgroups, p, stream);
}

}  // namespace

long experts_grad_workgroups(int out, int R, int E, int M, int N) { return (grad_plan(out, R, E, M, N).tiles + 7) / 8 * 8 * E; }

int experts_grad_way(int out, int R, int E, int M, int N)
{
    const Plan8 plan = grad_plan(out, R, E, M, N);
    return (plan.rows + plan.columns) / 2;
}

hipError_t launch_experts_grad(int out, int d_format, const ExpertsGradArgs &a, hipStream_t stream)
{
    const Plan8 plan = grad_plan(out, a.R, a.E, a.M, a.N);
    ExpertTileParams p = {};
    static_cast<TileParams &>(p) = TileParams{a.qd, a.sd, a.qx, a.sx, a.w, a.M, a.N, a.KB, a.N, 0, (a.M + plan.rows - 1) / plan.rows, (a.N + plan.columns - 1) / plan.columns,
                                              plan.rows * plan.columns > 64 * 64 && streamed(out, a.w, (long)a.E * a.M * a.N, a.N)};
    p.offsets = a.offsets, p.E = a.E, p.x_rows = a.R;
    const long n = (plan.tiles + 7) / 8 * 8 * a.E;
    return d_format == 0 ? launch<0>(out, plan, n, p, stream) : launch<1>(out, plan, n, p, stream);
}

}  // namespace tab
