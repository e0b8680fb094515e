// Gradients of the experts' weights: dW[e] = sum over the rows r of expert e of dY[r]^T X[r], from both operands packed along the rows by blocks of 128 that
// belong to one expert.  Every expert has the same tiles, and a tile goes through its expert's own blocks.
#include "tab_linear8_tiles.h"

namespace tab {

namespace {

Plan8 grad_plan(int out, int R, int E, int M, int N)
{
    constexpr TileTimes kFast[] = {{64, 64, 3, 0.05, 0.174, 0.8}, {64, 128, 2, 0.171, 0.242, 1.37}, {128, 128, 2, 0.571, 0.473, 1.69}, {256, 256, 1, 1.235, 1.125, 6.25}};
    constexpr TileTimes kExact[] = {{64, 64, 3, 0.371, 0.242, 0.7}, {64, 128, 2, 0.553, 0.336, 1.32}, {128, 128, 2, 1.22, 0.716, 1.65}};
    const int active = E < R ? E : R;
    const double steps = (double)R / active / kBlock8 + 0.5;
    Plan8 best = {};
    double least = 1e30;
    for (int i = 0; i < (out == 0 ? 3 : 4); i++) {
        const TileTimes &tile = out == 0 ? kExact[i] : kFast[i];
        const long tiles = ((M + (long)tile.rows - 1) / tile.rows) * ((N + (long)tile.columns - 1) / tile.columns);
        const double each = __builtin_ceil((double)tiles * active / 256), rounds = __builtin_ceil(each / tile.held);
        const double alone = tile.alone * rounds, among = tile.among * each;
        const double t = steps * (alone > among ? alone : among) + tile.out * each * (out == 0 ? 2 : 1);
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

long experts_grad_workgroups(int out, int R, int E, int M, int N) { return grad_plan(out, R, E, M, N).tiles * E; }

hipError_t launch_experts_grad(int out, int d_format, const ExpertsGradArgs &a, hipStream_t stream)
{
    const Plan8 plan = grad_plan(out, a.R, a.E, a.M, a.N);
    ExpertTileParams p = {};
    static_cast<TileParams &>(p) = TileParams{a.qd, a.sd, a.qx, a.sx, a.w, a.M, a.N, a.KB, a.N, 0, (a.M + plan.rows - 1) / plan.rows, (a.N + plan.columns - 1) / plan.columns};
    p.offsets = a.offsets, p.E = a.E, p.x_rows = a.R;
    return d_format == 0 ? launch<0>(out, plan, plan.tiles * a.E, p, stream) : launch<1>(out, plan, plan.tiles * a.E, p, stream);
}

}  // namespace tab
