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
                                              (int)run_tiles_most(a.R, a.E, plan.rows), (a.N + plan.columns - 1) / plan.columns,
                                              plan.parts == 1 && plan.rows * plan.columns > 64 * 64 && streamed(out, a.y, (long)a.R * a.N, a.N)};
    p.offsets = a.offsets, p.rows = a.rows, p.E = a.E, p.x_rows = a.x_rows;
    if (plan.parts == 1 && out != 0)
        return out == 1 ? launch_expert_tiles<FORMAT, 1, false, WBITS>(plan, p, stream) : launch_expert_tiles<FORMAT, 2, false, WBITS>(plan, p, stream);
    const hipError_t e = out == 0 && full_sums ? launch_expert_tiles<FORMAT, 0, true, WBITS>(plan, p, stream) : launch_expert_tiles<FORMAT, 0, false, WBITS>(plan, p, stream);
    return e != hipSuccess || plan.parts == 1 ? e : launch_join(out, static_cast<const float *>(workspace), a.y, (long)a.R * a.N, plan.parts, stream);
}

// Few rows to an expert: bound by reading the weights of the experts that are chosen.  A workgroup takes at most 2^log_most rows of an expert and some groups of
// 16 rows of its weight, `split` waves to a group, which take its blocks of K in turn, 2 * AHEAD of them on their way in every wave.  The rows of X lie in
// LDS, as in linear8_rows.  What a small call takes is the way to the weights: the expert, its rows' numbers, the rows, each a round trip to memory, so
// the first blocks of the weight are asked for as soon as the expert is known.  60 rows, 24 experts of 1003 x 776, fp16: 8.0 us (a quantizer and tiles 18.7); 64 rows, 64
// experts of 2048 x 4096, 4 bits: 29 us, 184 MB at 6.2 TB/s.
struct ExpertRowsParams {
    const void *x;
    const uint8_t *sx, *qw, *sw;
    void *y;
    const int *offsets, *rows;
    int M, N, K, KB, w_scale_rows, E, x_rows, each, split, log_most;  // each: workgroups to a run of rows
    long ldx;
    Div32 div_kb;
};

template <int INPUT, int FORMAT, int OUT, int WBITS>
__global__ __launch_bounds__(64 * kRowsWaves) __attribute__((amdgpu_waves_per_eu(4))) void experts_rows(const ExpertRowsParams p)
{
    using T = typename Element<OUT>::type;
    using X = typename Element<INPUT == 3 ? 0 : INPUT>::type;
    constexpr int WAVES = kRowsWaves, AHEAD = 4, kWBlock = kBlock8 * WBITS / 8;
    extern __shared__ __attribute__((aligned(16))) uint8_t packed[];
    __shared__ __attribute__((aligned(16))) float sums[WAVES * 256];
    const int t = threadIdx.x, lane = t % 64, wave = __builtin_amdgcn_readfirstlane(t / 64), l16 = lane % 16, quarter = lane / 16;
    const int place = (int)blockIdx.x / p.each, share = (int)blockIdx.x - place * p.each;
    const Run run = find_run(p.offsets, p.E, p.M, (uint32_t)place, p.log_most, lane);
    if (run.expert < 0) return;
    const int first_row = run.first, rows = min(1 << p.log_most, run.end - first_row);
    const int sets = WAVES / p.split, part = wave % p.split, groups = (p.N + 15) / 16, group = share * sets + wave / p.split;
    if (run.expert == p.E) {  // rows of no expert: zeros
        const int n0 = share * sets * 16, columns = min(sets * 16, p.N - n0);
        for (int m = 0; m < rows; m++)
            for (int n = t; n < columns; n += 64 * WAVES) static_cast<T *>(p.y)[(long)(first_row + m) * p.N + n0 + n] = (T)0.f;
        return;
    }
    // the weight: the same place in every lane, and a lane's own from there
    const bool w_rows = p.w_scale_rows == p.N;
    const int w_row_bytes = p.KB * kWBlock, scale_step = p.w_scale_rows * (WBITS == 4 ? 4 : 1), stride = rows_stride(p.KB);
    const int n0 = min(group, groups - 1) * 16, row = min(l16, p.N - 1 - n0);
    const uint8_t *const w_at = p.qw + ((long)run.expert * p.N + n0) * w_row_bytes;
    const uint8_t *const s_at = p.sw + (long)run.expert * p.KB * scale_step + (WBITS == 4 ? n0 * 4 : w_rows ? n0 : n0 / kBlock8);
    const uint32_t w_lane = (uint32_t)(row * w_row_bytes + quarter * 16), s_lane = (uint32_t)(WBITS == 4 ? row * 4 + quarter : w_rows ? row : 0);
    // block i of a wave: every split-th one, or (of 4 bits) every split-th pair, which is a cache line
    auto block_of = [&](int i) { return WBITS == 4 ? (i / 2 * p.split + part) * 2 + i % 2 : i * p.split + part; };
    struct Blocks {
        i32x4 low[AHEAD], high[WBITS == 8 ? AHEAD : 1];
        uint32_t scale[AHEAD];
    };
    auto load = [&](Blocks &to, int i) {  // blocks i .. i + AHEAD - 1 of the wave
#pragma unroll
        for (int u = 0; u < AHEAD; u++) {
            const int kb = block_of(i + u);
            if (kb >= p.KB) continue;  // (the same for the whole wave)
            const uint8_t *const w = w_at + kb * kWBlock;
            to.low[u] = *reinterpret_cast<const i32x4 *>(w + w_lane);
            if constexpr (WBITS == 8) to.high[u] = *reinterpret_cast<const i32x4 *>(w + w_lane + 64);
            to.scale[u] = (s_at + (long)kb * scale_step)[s_lane];
        }
    };
    Blocks even, odd;
    load(even, 0);
    load(odd, AHEAD);

    // X into LDS: 16 lanes a block
    constexpr int AT_ONCE = sizeof(X) == 4 && INPUT != 3 ? 2 : 4, STEP = 64 * WAVES / 16;
    uint32_t *const scales = reinterpret_cast<uint32_t *>(packed + rows * stride);
    const int blocks = rows * p.KB;
#pragma nounroll
    for (int first = t / 16; first < blocks; first += AT_ONCE * STEP) {
        Words<X> v[AT_ONCE];
#pragma unroll
        for (int u = 0; u < AT_ONCE; u++) {
            const int block = min(first + u * STEP, blocks - 1), m = (int)div32(block, p.div_kb), kb = block - m * p.KB;
            const int from = p.rows ? p.rows[first_row + m] : first_row + m;
            const bool there = from >= 0 && from < p.x_rows;
            if constexpr (INPUT == 3) {
                v[u] = {};
                if (there) {
                    const uint2 w = *reinterpret_cast<const uint2 *>(static_cast<const uint8_t *>(p.x) + ((long)from * p.KB + kb) * kBlock8 + l16 * 8);
                    v[u].w[0] = w.x, v[u].w[1] = w.y, v[u].w[2] = p.sx[(long)kb * p.x_rows + from];
                }
            } else {
                v[u] = load_words(static_cast<const X *>(p.x) + from * p.ldx, kb * kBlock8 + l16 * 8, there ? p.K : 0);
            }
        }
#pragma unroll
        for (int u = 0; u < AT_ONCE; u++) {
            const int block = first + u * STEP, m = (int)div32(block, p.div_kb), kb = block - m * p.KB;
            if (block >= blocks) break;
            uint32_t byte;
            uint2 w;
            if constexpr (INPUT == 3) w = {v[u].w[0], v[u].w[1]}, byte = v[u].w[2];
            else w = pack_run<X, FORMAT>(v[u], byte);
            *reinterpret_cast<uint2 *>(packed + m * stride + kb * kBlock8 + l16 * 8) = w;
            if (l16 == 0) scales[kb * rows + m] = byte;
        }
    }
    __syncthreads();

    const int m = min(l16, rows - 1);  // (columns past the last row repeat it and are not stored)
    const uint8_t *const x_row = packed + m * stride;
    f32x4 acc = {0.f, 0.f, 0.f, 0.f};
    auto multiply = [&](const Blocks &of, int i) {
#pragma unroll
        for (int u = 0; u < AHEAD; u++) {
            const int kb = block_of(i + u);
            if (kb >= p.KB) continue;
            acc = times_rows<FORMAT, OUT, WBITS>(w_numbers<WBITS>(of.low[u], of.high[WBITS == 8 ? u : 0]), of.scale[u], x_row + kb * kBlock8, scales[kb * rows + m], quarter, acc);
        }
    };
    if (group < groups) {
        for (int i = 0;; i += 2 * AHEAD) {
            const bool more = block_of(i + 2 * AHEAD) < p.KB;
            multiply(even, i);
            if (more) load(even, i + 2 * AHEAD);
            multiply(odd, i + AHEAD);
            if (!more) break;
            load(odd, i + 3 * AHEAD);
        }
    }
    if (p.split > 1) {  // the waves' parts in their order
        *reinterpret_cast<f32x4 *>(sums + wave * 256 + lane * 4) = acc;
        __syncthreads();
        if (part == 0)
            for (int k = 1; k < p.split; k++) acc += *reinterpret_cast<const f32x4 *>(sums + (wave + k) * 256 + lane * 4);
    }
    const int n = group * 16 + quarter * 4;
    if (part != 0 || l16 >= rows || n >= p.N) return;
    T *const to = static_cast<T *>(p.y) + (long)(first_row + l16) * p.N + n;
    if (n + 4 <= p.N) {
        store4(to, acc);
    } else {
        for (int e = 0; e < 4; e++)
            if (n + e < p.N) to[e] = (T)acc[e];
    }
}

template <int INPUT, int FORMAT, int OUT, int WBITS> hipError_t launch_expert_rows(const ExpertsPlan &plan, const ExpertsArgs &a, int scale_rows, hipStream_t stream)
{
    const ExpertRowsParams p = {a.x, a.sx, a.qw, a.sw, a.y, a.offsets, a.rows, a.R, a.N, a.K, a.KB, scale_rows, a.E, a.x_rows, (a.N + plan.columns - 1) / plan.columns, plan.parts,
                                log2_of(plan.rows), a.ldx, make_div32((uint32_t)a.KB)};
    experts_rows<INPUT, FORMAT, OUT, WBITS><<<(unsigned)plan.workgroups, 64 * kRowsWaves, (unsigned)rows_lds(plan.rows, a.KB), stream>>>(p);
    return hipGetLastError();
}

template <int WBITS> hipError_t launch_expert_few(int dtype, const ExpertsPlan &plan, const ExpertsArgs &a, int scale_rows, hipStream_t stream)
{
    return dtype == 0 ? launch_expert_rows<0, 0, 0, WBITS>(plan, a, scale_rows, stream)
                      : dtype == 1 ? launch_expert_rows<1, 0, 1, WBITS>(plan, a, scale_rows, stream) : launch_expert_rows<2, 0, 2, WBITS>(plan, a, scale_rows, stream);
}

}  // namespace

}  // namespace tab
