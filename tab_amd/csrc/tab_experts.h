// Rows sorted by expert: the runs of rows that `offsets` cuts out, and their tiles, as a kernel finds them.  Expert e has the rows offsets[e] ..
// offsets[e + 1]; what is behind offsets[E] belongs to no expert.  The numbers are on the device alone, so a launch has as many workgroups as
// there can be tiles, and every wave looks its own tile up: 64 experts a step, a few hundred cycles at the most for the first 64 (most of it one
// load), which costs less than a launch that lays tables of tiles out.  Offsets that are not in order, or not between 0 and `rows`,
// are cut to what is: no access depends on them being right.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace tab {

constexpr int kExpertsMost = 1024;
constexpr int kRunBlock = 128;  // rows of a block of the gradients of weights: every expert's rows begin at a new one

// Blocks of kRunBlock rows that `rows` rows in E runs take at most
__host__ __device__ inline int run_blocks_most(int rows, int E) { return (int)(((long)rows + (kRunBlock - 1) * (long)(E < rows ? E : rows)) / kRunBlock); }
// Tiles of `tile` rows that they take at most, those behind the last expert included
inline long run_tiles_most(int rows, int E, int tile) { return ((long)rows + (tile - 1) * (E + 1L < rows ? E + 1L : (long)rows)) / tile; }

struct Run { int expert, first, end; };  // expert E: behind the last one; -1: none

// Sum over this lane and those below it
__device__ __forceinline__ int wave_scan(int v)
{
    v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, false);  // of the lanes 1, 2, 4, 8 below in a row of 16
    v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, false);  // the last of row 0 to row 1, of 2 to 3,
    v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, false);  // the last of row 1 to rows 2 and 3
    return v;
}

// Rows a .. b of expert e (of E: those behind the last; past E: none)
__device__ __forceinline__ void run_bounds(const int *offsets, int E, int rows, int e, int &a, int &b)
{
    a = e <= E ? min(max(offsets[e], 0), rows) : rows;
    b = e < E ? min(max(offsets[e + 1], a), rows) : rows;
}
// Tiles of 2^log_tile rows
__device__ __forceinline__ int run_tiles(int a, int b, int log_tile) { return (int)(((uint32_t)(b - a) + (1u << log_tile) - 1u) >> log_tile); }
constexpr int log2_of(int n) { return n > 1 ? 1 + log2_of(n / 2) : 0; }

// Tiles of all runs, with or without those behind the last expert.  By whole waves.
__device__ __forceinline__ uint32_t count_runs(const int *offsets, int E, int rows, bool behind, int log_tile, int lane)
{
    uint32_t all = 0;
    const int last = behind ? E : E - 1;
    for (int base = 0; base <= last; base += 64) {
        int a, b;
        run_bounds(offsets, E, rows, base + lane, a, b);
        all += (uint32_t)__builtin_amdgcn_readlane(wave_scan(base + lane <= last ? run_tiles(a, b, log_tile) : 0), 63);
    }
    return all;
}

// Tile `id`: its expert, its first row and the end of the expert's rows.  By whole waves.
__device__ __forceinline__ Run find_run(const int *offsets, int E, int rows, uint32_t id, int log_tile, int lane)
{
    uint32_t before = 0;
    for (int base = 0; base <= E; base += 64) {
        int a, b;
        run_bounds(offsets, E, rows, base + lane, a, b);
        const int mine = run_tiles(a, b, log_tile), sum = wave_scan(mine);
        const uint64_t past = __ballot(before + (uint32_t)sum > id);
        if (past) {
            const int l = __builtin_ctzll(past);
            const uint32_t first = before + (uint32_t)(__builtin_amdgcn_readlane(sum, l) - __builtin_amdgcn_readlane(mine, l));
            return {base + l, __builtin_amdgcn_readlane(a, l) + (int)((id - first) << log_tile), __builtin_amdgcn_readlane(b, l)};
        }
        before += (uint32_t)__builtin_amdgcn_readlane(sum, 63);
    }
    return {-1, 0, 0};
}

// Expert e's blocks of 2^log_tile rows, where every expert's rows begin at a new one: first and end.  By whole waves.
__device__ __forceinline__ Run run_of(const int *offsets, int E, int rows, int expert, int log_tile, int lane)
{
    int before = 0;
    for (int base = 0;; base += 64) {
        int a, b;
        run_bounds(offsets, E, rows, base + lane, a, b);
        const int mine = run_tiles(a, b, log_tile), sum = wave_scan(mine);
        if (expert < base + 64) {
            const int end = before + __builtin_amdgcn_readlane(sum, expert - base);
            return {expert, end - __builtin_amdgcn_readlane(mine, expert - base), end};
        }
        before += __builtin_amdgcn_readlane(sum, 63);
    }
}

// ---- launchers (tab_experts8.hip, tab_experts4.hip, tab_experts_grad.hip, tab_route.hip, tab_combine.hip) -----------------------------

// Y[r] = X[rows[r]] QW[e]^T for the rows r of expert e; rows null: X[r]
struct ExpertsArgs {
    const void *x;                  // packed numbers, or elements of Y's type
    const uint8_t *sx, *qw, *sw;    // sx: of packed numbers
    void *y;
    const int *offsets, *rows;
    int x_rows, R, E, N, K, KB;
    int w_block_rows;               // 8 bits: rows of QW under one scale, 1 or 128
    long ldx;                       // elements between rows of x that are not packed
};
// How a call is computed: few rows to an expert quantized and multiplied in one launch, or tiles of a packed X, K in parts
struct ExpertsPlan {
    bool few;
    int rows, columns;              // of a tile; few: rows of X in a workgroup's LDS (a power of two) and of the weight that it takes
    int parts, kb_per_part;         // few: waves that share 16 rows of the weight, and 0
    long workgroups;
};
ExpertsPlan experts_plan(int out_dtype, bool full_sums, int bits, int R, int E, int N, int KB);
// full_sums: of an fp32 Y, as of one from fp32 activations; else those towards 16 bits
hipError_t launch_experts8(int out_dtype, bool full_sums, int x_format, const ExpertsPlan &plan, const ExpertsArgs &a, void *workspace, hipStream_t stream);
hipError_t launch_experts4(int out_dtype, const ExpertsPlan &plan, const ExpertsArgs &a, void *workspace, hipStream_t stream);
hipError_t launch_experts8_few(int dtype, const ExpertsPlan &plan, const ExpertsArgs &a, hipStream_t stream);
hipError_t launch_experts4_few(int dtype, const ExpertsPlan &plan, const ExpertsArgs &a, hipStream_t stream);

// W[e] (M x N) = QD[:, e's blocks] QX[:, e's blocks]^T, both operands packed along the rows by expert (M and N x blocks)
struct ExpertsGradArgs {
    const uint8_t *qd, *sd, *qx, *sx;
    void *w;
    const int *offsets;
    int R, E, M, N, KB;
};
long experts_grad_workgroups(int out_dtype, int R, int E, int M, int N);
int experts_grad_way(int out_dtype, int R, int E, int M, int N);  // (the tile's rows + columns) / 2
hipError_t launch_experts_grad(int out_dtype, int d_format, const ExpertsGradArgs &a, hipStream_t stream);

struct RouteArgs {
    const void *logits;
    float *weights;
    int *experts, *rows, *places, *offsets, *workspace;
    long ld;
    int M, E, k;
    bool normalize;
};
constexpr int kChoicesMost = 32;
size_t route_workspace(int M, int E, int k);
hipError_t launch_route(int dtype, const RouteArgs &a, hipStream_t stream);

struct RouteGradArgs {
    const float *dweights, *weights;
    const int *experts;
    const void *logits;
    void *dlogits;
    long ld;
    int M, E, k;
    bool normalize;
};
hipError_t launch_route_grad(int dtype, const RouteGradArgs &a, hipStream_t stream);

struct CombineArgs {
    const void *y;
    const int *places;
    const float *weights;           // null: ones
    void *out;
    int M, k, R, D;
};
hipError_t launch_combine(int y_dtype, int out_dtype, const CombineArgs &a, hipStream_t stream);  // out_dtype: y_dtype, or y_dtype fp32

struct CombineGradArgs {
    const void *dout, *y;
    const int *places, *used;       // used: rows of Y that belong to a token; null: all
    const float *weights;           // null: ones
    void *dy;                       // null: not wanted
    float *dweights;                // null: not wanted
    int M, k, R, D;
};
hipError_t launch_combine_grad(int dtype, const CombineGradArgs &a, hipStream_t stream);

}  // namespace tab
