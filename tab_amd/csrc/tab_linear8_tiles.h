// Product of two packed 8-bit operands with power-of-two scales per block of 128,
//   Y[m][n] = sum over kb of 2^(SX[kb][m] + SW[kb][n] - 254) * sum over k in block kb of QX[m][k] QW[n][k].
//
// 16-bit outputs: v_mfma_scale_f32_16x16x128_f8f6f4.  One instruction is a 16 x 16 tile over one block of K, and it takes the E8M0 bytes of its
// 16 rows and 16 columns as operands, so the scales cost no vector instruction and the sums stay in one set of fp32 accumulators.  Inside
// the instruction, products of eight neighbours in K are aligned to the largest of them and keep 13 bits below it (measured): 1.5e-5 of the
// output's size for normal operands, far below the 2^-8 or 2^-11 of the output's own rounding, but not what an fp32 output is for.  (Outputs that are the other
// neighbour of what full sums round to: 0.5-1.7 % in bf16, 3-7 % in fp16.  Off the exact product, of its size: 512 x 4096 x 4096 bf16 0.0016633 instead of 0.0016632,
// K = 776 fp16 0.0002077 instead of 0.0002070.  The same call gives the same bits.)
// fp32 outputs (EXACT): the numbers times their scales are bf16 numbers exactly (4 of 8 significant bits, the exponent range of fp32), made by one
// conversion of two numbers, and v_mfma_f32_16x16x32_bf16 multiplies them at half the rate with full fp32 sums.  A number below 2^-126 may
// count as zero there.
#pragma once
#include "tab_blocks8.h"
#include "tab_common.h"
#include "tab_experts.h"

namespace tab {

namespace {

typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

constexpr int kBufferFlags8 = 0x00020000;     // descriptor word 3: untyped 32-bit data

struct TileParams {
    const uint8_t *qx, *sx, *qw, *sw;
    void *y;
    int M, N, KB, w_scale_rows;  // w_scale_rows: scales of QW per block of K, N or ceil(N / 128)
    int kb_per_part;             // blocks of K of a part; with more than one part y is [parts][M][N] fp32
    int tiles_m, tiles_n;
    int streamed;                // y is written past the caches (see streamed())
};

// A launch over the experts of a layer.  Rows (kRowsByExpert): row r of Y belongs to the expert e with offsets[e] <= r < offsets[e + 1], is multiplied by
// QW[e] (N x K) and comes from row rows[r] of X, or r; rows behind the last expert's become zeros.  K (kKByExpert): Y[e] (M x N) is the product over
// the expert's own run of blocks of K.
constexpr int kOneWeight = 0, kRowsByExpert = 1, kKByExpert = 2;
struct ExpertTileParams : TileParams {
    const int *offsets, *rows;
    int E, x_rows;  // kRowsByExpert: rows of X; kKByExpert: rows that offsets cuts up
};
template <int BY> struct TileParamsOf { using type = ExpertTileParams; };
template <> struct TileParamsOf<kOneWeight> { using type = TileParams; };

// WBITS: 8, E4M3, or 4, E2M1 (the instruction's format 4)
template <int FORMAT, int WBITS = 8> __device__ __forceinline__ f32x4 mfma16(i32x8 w, i32x8 x, f32x4 c, uint32_t w_scale, uint32_t x_scale)
{
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(w, x, c, WBITS == 4 ? 4 : 0, FORMAT, 0, (int)w_scale, 0, (int)x_scale);
}

// A lane's 32 numbers of a block times their scale, exactly
struct Exact32 { bf16x8 v[4]; };

template <int FORMAT> __device__ __forceinline__ Exact32 exact32(i32x8 q, uint32_t scale_byte)
{
    const float scale = __uint_as_float(scale_byte << 23);
    Exact32 e;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        bf16x2 p[4];
#pragma unroll
        for (int j = 0; j < 2; j++) {
            if constexpr (FORMAT == 0) {
                p[2 * j] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(q[2 * i + j], scale, false);
                p[2 * j + 1] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(q[2 * i + j], scale, true);
            } else {
                p[2 * j] = __builtin_amdgcn_cvt_scalef32_pk_bf16_bf8(q[2 * i + j], scale, false);
                p[2 * j + 1] = __builtin_amdgcn_cvt_scalef32_pk_bf16_bf8(q[2 * i + j], scale, true);
            }
        }
        e.v[i] = bf16x8{p[0][0], p[0][1], p[1][0], p[1][1], p[2][0], p[2][1], p[3][0], p[3][1]};
    }
    return e;
}

// The same of a lane's 32 numbers of 4 bits; a scale byte of 255 is NaN
__device__ __forceinline__ Exact32 exact32_of4(i32x8 q, uint32_t scale_byte)
{
    const float scale = __uint_as_float(scale_byte << 23 | (scale_byte == 255u ? 0x400000u : 0u));
    Exact32 e;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const bf16x2 p[4] = {__builtin_amdgcn_cvt_scalef32_pk_bf16_fp4((uint32_t)q[i], scale, 0), __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4((uint32_t)q[i], scale, 1),
                             __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4((uint32_t)q[i], scale, 2), __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4((uint32_t)q[i], scale, 3)};
        e.v[i] = bf16x8{p[0][0], p[0][1], p[1][0], p[1][1], p[2][0], p[2][1], p[3][0], p[3][1]};
    }
    return e;
}

__device__ __forceinline__ f32x4 mfma16_exact(const Exact32 &w, const Exact32 &x, f32x4 c)
{
#pragma unroll
    for (int i = 0; i < 4; i++) c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(w.v[i], x.v[i], c, 0, 0, 0);
    return c;
}

// Global memory straight into LDS: 16 bytes a lane at `to` + 16 * lane, or one byte a lane, zero-extended, at `to` + 4 * lane.  A lane offset at or
// past the end of the buffer gives zeros.  In assembly because of the waits that the compiler puts around the builtin: it has a wave that
// reads LDS wait for all its loads on the way there, which leaves one step of K in flight at most; here wait_loads counts them.
// (m0 may not be used by the instruction after its write, nor a scalar register by a memory instruction in the five after a vector
// instruction's write.)
__device__ __forceinline__ void to_lds16(i32x4 buffer, uint32_t to, uint32_t lane_offset)
{
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 4\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds" ::"s"(to), "v"(lane_offset), "s"(buffer) : "memory", "m0");
}
__device__ __forceinline__ void to_lds1(i32x4 buffer, uint32_t to, uint32_t lane_offset)
{
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 4\n\tbuffer_load_ubyte %1, %2, 0 offen lds" ::"s"(to), "v"(lane_offset), "s"(buffer) : "memory", "m0");
}
__device__ __forceinline__ void to_lds4(i32x4 buffer, uint32_t to, uint32_t lane_offset)  // a word a lane
{
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 4\n\tbuffer_load_dword %1, %2, 0 offen lds" ::"s"(to), "v"(lane_offset), "s"(buffer) : "memory", "m0");
}
__device__ __forceinline__ uint32_t lds_address(const uint8_t *p) { return (uint32_t)(uintptr_t)(const __attribute__((address_space(3))) uint8_t *)p; }

// A buffer of `bytes` (below 2^31; none if negative) from p on, the same in every lane: base, size, flags
__device__ __forceinline__ i32x4 buffer(const uint8_t *p, int bytes)
{
    const uint64_t at = (uint64_t)p;
    return i32x4{__builtin_amdgcn_readfirstlane((int)(uint32_t)at), __builtin_amdgcn_readfirstlane((int)(at >> 32) & 0xffff),
                 __builtin_amdgcn_readfirstlane(max(bytes, 0)), kBufferFlags8};
}
// The rows that are gathered are one buffer of up to this many bytes; an offset from here on, with less than 2^28 added, is past its end
constexpr uint32_t kGatherMost = 0xe0000000u;

// This wave's loads but for the last `behind` have landed (s_waitcnt's vmcnt alone; bits 3:0 and 15:14)
template <int BEHIND> __device__ __forceinline__ void wait_loads() { __builtin_amdgcn_s_waitcnt(0x0f70 | (BEHIND & 15) | (BEHIND >> 4) << 14); }

template <int N> struct ScaleWords { uint32_t w[N]; };  // the scales of a lane's N groups of 16 rows

template <int N> __device__ __forceinline__ ScaleWords<N> scale_words(const uint32_t *p)
{
    ScaleWords<N> s;
    if constexpr (N % 4 == 0) {
#pragma unroll
        for (int i = 0; i < N / 4; i++) {
            const uint4 v = reinterpret_cast<const uint4 *>(p)[i];
            s.w[4 * i] = v.x, s.w[4 * i + 1] = v.y, s.w[4 * i + 2] = v.z, s.w[4 * i + 3] = v.w;
        }
    } else {
        static_assert(N == 2, "groups of 16 rows of a wave");
        const uint2 v = *reinterpret_cast<const uint2 *>(p);
        s.w[0] = v.x, s.w[1] = v.y;
    }
    return s;
}

template <typename T> __device__ __forceinline__ void store4(T *y, f32x4 v)
{
    struct __attribute__((packed, aligned(sizeof(T)))) Four { T v[4]; };
    *reinterpret_cast<Four *>(y) = Four{{(T)v[0], (T)v[1], (T)v[2], (T)v[3]}};
}

// A workgroup of WM x WN waves makes a BM x BN tile of Y, for more rows than linear8_rows takes; bound by the matrix instructions and, the smaller the tile,
// by the way of its operands into LDS (54 bytes a clock and CU measured; reads of LDS reach 200).  What cost most was a wave that waits to get a load
// out, or whose scalar instructions make the load's address, and does not multiply meanwhile.  So a step's operands are read from LDS while the
// step before is multiplied, loads, reads and products alternate, and a load takes two scalar instructions and one addition.
//   256 x 256  8192^3 363 us, 3.03 PFLOP/s, in a replayed graph, its output past the caches (404-406 through them; 389 with X's quantizer; a library's fp8 product
//              with one scale a tensor 361); weights of 4 bits 332
//   128 x 128  4096 x 2048 x 4096 33 us, 2.1 PFLOP/s
//   64 x 128   512 x 4096 x 4096 13.8 us, 1.25 PFLOP/s (64 x 64 16.4; both 19 with read and multiplied in turn)
//   64 x 64    128 x 4096 x 4096 9.0 us (14.0 in turn); fp32 1000 x 776 x 520 6.6 us
// A step is one block of K: 128 bytes of each of the tile's rows and their scales,
// straight from global memory into one of STAGES parts of LDS.  A row is eight pieces of 16 bytes; row r has piece g at place g ^ (r & 7), so
// that lanes that read at once meet different banks.  Which piece a lane multiplies is free as long as both operands agree, since a block
// has one scale.
//
// Weights of 4 bits (WBITS 4): a row's block is 64 bytes, four pieces, row r's piece g at place g ^ (r >> 2 & 3); lane (row, quarter) multiplies the
// quarter-th 32 numbers of the block, one group, whose scale is byte `quarter` of the row's word.  (Products in bf16 take X's numbers in the same order.)
template <int BM, int BN, int WM, int WN, int STAGES, int FORMAT, int OUT, bool EXACT, int WBITS = 8, int BY = kOneWeight>
__global__ __launch_bounds__(64 * WM * WN, 2) void linear8_tiles(const typename TileParamsOf<BY>::type p)
{
    using T = typename Element<OUT>::type;
    constexpr int WAVES = WM * WN, THREADS = 64 * WAVES, TM = BM / WM / 16, TN = BN / WN / 16;
    constexpr int kWBlock = kBlock8 * WBITS / 8, W_LANES = kWBlock / 16, W_ROWS = 64 / W_LANES;  // bytes of a row's block; lanes a row and rows of one load
    constexpr int NUMBERS = BM * kBlock8 + BN * kWBlock, STAGE = NUMBERS + 4 * THREADS;
    constexpr int W_WAVES = WAVES == 8 ? WN : WAVES;  // of eight waves the first four load W and the scales
    constexpr int A_LOADS = BM / 8 / WAVES, W_LOADS = BN / W_ROWS / W_WAVES, LOADS = A_LOADS + W_LOADS;
    constexpr bool GATHER = BY == kRowsByExpert;
    static_assert(BM + BN <= THREADS, "a lane loads one scale");
    __shared__ __attribute__((aligned(1024))) uint8_t lds[STAGES * STAGE];

    // the tile: parts of K outermost; every XCD (workgroup number modulo 8) takes one run of the tiles, and a run goes through
    // groups of 8 tiles of rows, so that what its CUs hold at one time reads few rows of either operand
    // (over experts p.tiles_m is a bound, and the workgroups past the tiles that there are have nothing to do)
    const int t = threadIdx.x, lane = t % 64;
    const uint32_t most = (uint32_t)p.tiles_m * (uint32_t)p.tiles_n, part = blockIdx.x / most, b = blockIdx.x - part * most;
    uint32_t all_m = (uint32_t)p.tiles_m;
    if constexpr (BY == kRowsByExpert) {
        all_m = count_runs(p.offsets, p.E, p.M, true, log2_of(BM), lane);
        if (b >= all_m * (uint32_t)p.tiles_n) return;
    }
    const uint32_t tiles = all_m * (uint32_t)p.tiles_n;
    uint32_t share = tiles / 8, id = b, expert = 0;
    if constexpr (BY == kKByExpert) {
        // every XCD takes an eighth of each expert's tiles (the experts' runs of blocks differ, and with them their tiles' times), rounded up
        share = (most + 7) / 8;
        expert = blockIdx.x / (share * 8);
        id = blockIdx.x - expert * (share * 8);
        id = (id & 7) * share + (id >> 3);
        if (id >= most) return;
    } else if (id < share * 8) {
        id = (id & 7) * share + (id >> 3);
    }
    const uint32_t in_group = 8 * (uint32_t)p.tiles_n, group = id / in_group, rest = id - group * in_group;
    const uint32_t rows = min(8u, all_m - group * 8), tile_n = rest / rows, tile_m = group * 8 + rest - tile_n * rows;
    int m0 = (int)tile_m * BM, end_m = p.M;
    const int n0 = (int)tile_n * BN;
    int kb0 = (int)part * p.kb_per_part, kb1 = min(p.KB, kb0 + p.kb_per_part);
    if constexpr (BY == kRowsByExpert) {
        const Run run = find_run(p.offsets, p.E, p.M, tile_m, log2_of(BM), lane);
        if (run.expert < 0) return;  // (offsets out of order, the count of their tiles past 32 bits)
        expert = (uint32_t)run.expert, m0 = run.first, end_m = run.end;
        if (run.expert == p.E) expert = 0, kb1 = kb0;  // rows of no expert: zeros
    }
    if constexpr (BY == kKByExpert) {
        const Run run = run_of(p.offsets, p.E, p.x_rows, (int)expert, log2_of(kRunBlock), lane);
        kb0 = (int)min((uint32_t)run.first, (uint32_t)p.KB), kb1 = max(kb0, (int)min((uint32_t)run.end, (uint32_t)p.KB));  // (whatever offsets holds)
    }

    // Every expert begins at another block of K: rows of 4096 numbers are as many bytes apart, so that all tiles at the same block would ask the same few
    // channels of the memory (32 experts of 2048 x 4096, 512 rows each: 149 us, now 127)
    const int turn = BY == kRowsByExpert && p.kb_per_part == p.KB ? (int)expert % p.KB : 0;

    const int wave = __builtin_amdgcn_readfirstlane(t / 64), wm = wave / WN, wn = wave % WN, l16 = lane % 16, quarter = lane / 16;
    const int row_bytes = p.KB * kBlock8, w_row_bytes = p.KB * kWBlock, rows_x = min(BM, end_m - m0), rows_w = min(BN, p.N - n0);
    // one buffer holds X: listed rows from the first one on, as a list may name any, others from the tile's
    int x_first = m0;
    if constexpr (GATHER) x_first = p.rows ? 0 : m0;
    const uint8_t *const qx = p.qx + (long)x_first * row_bytes;
    const uint8_t *const qw = p.qw + ((BY == kRowsByExpert ? (long)expert * p.N : 0) + n0) * (long)w_row_bytes;
    const uint8_t *const sw = p.sw + (BY == kRowsByExpert ? (long)expert * p.KB * p.w_scale_rows * (WBITS == 4 ? 4 : 1) : 0);
    // load i of a wave is eight rows of an operand's tile, eight lanes a row: of W the waves take turns, of X those that multiply the rows
    const int first_x = wm * (BM / WM) + wn * 8, first_w = wave * W_ROWS;
    const uint32_t x_at = (uint32_t)(first_x + lane / 8) * (uint32_t)row_bytes + (uint32_t)((lane % 8) ^ (lane / 8)) * 16;
    uint32_t w_at = (uint32_t)(first_w + lane / W_LANES) * (uint32_t)w_row_bytes + (uint32_t)(turn * kWBlock) +
                    (uint32_t)(WBITS == 4 ? (lane % 4) ^ (lane / 16) : (lane % 8) ^ (lane / 8)) * 16;
    // row `row` of the tile in the buffer of X, in units of `unit` bytes
    auto gathered = [&](int row, int unit) {
        if constexpr (GATHER) {
            if (row >= rows_x) return kGatherMost;
            const int from = p.rows ? p.rows[m0 + row] : row;
            return from >= 0 && from < p.x_rows - x_first ? (uint32_t)from * (uint32_t)unit : kGatherMost;
        }
        return 0u;
    };
    uint32_t x_from[GATHER ? A_LOADS : 1];
    if constexpr (GATHER) {
#pragma unroll
        for (int i = 0; i < A_LOADS; i++) x_from[i] = gathered(first_x + i * 8 * WN + lane / 8, row_bytes) + (uint32_t)(turn * kBlock8) + (uint32_t)((lane % 8) ^ (lane / 8)) * 16;
    }
    // A lane loads one scale: place t of X's, then of W's (of eight waves the first four load one of each).  The scales of a lane's groups of 16 rows are
    // side by side.  (A wave's scales are all of X or all of W.)
    const bool row_scales = p.w_scale_rows == p.N;
    const int first = kb0 + turn;
    struct Scales { const uint8_t *at; int step, rows; uint32_t offset; };
    auto scales_of = [&](bool x, int place, bool any) {
        const int groups = x ? TM : TN, row = place / (16 * groups) * (16 * groups) + place % groups * 16 + place / groups % 16;
        if constexpr (GATHER)
            if (x) return Scales{p.sx + x_first + (long)first * p.x_rows, p.x_rows, !any ? 0 : p.x_rows - x_first, gathered(row, 1)};
        if (WBITS == 4 && !x) return Scales{sw + ((long)first * p.N + n0) * 4, p.N * 4, any ? rows_w * 4 : 0, (uint32_t)row * 4};
        const int step = x ? p.M : p.w_scale_rows;
        return Scales{(x ? p.sx + m0 : sw + (row_scales ? n0 : n0 / kBlock8)) + (long)first * step, step,
                      !any ? 0 : x ? rows_x : row_scales ? rows_w : (n0 + rows_w - 1) / kBlock8 - n0 / kBlock8 + 1,
                      (uint32_t)(x || row_scales ? row : (n0 + row) / kBlock8 - n0 / kBlock8)};
    };
    const bool scale_x = WAVES == 8 || wave * 64 < BM;
    Scales scales = scales_of(scale_x, scale_x ? t : t - BM, wave * 64 < BM + BN), more_scales = scales_of(false, t, true);
    const uint32_t lds_at = lds_address(lds);
    // the rows of an operand's tile are one buffer: rows past its end, and with a size of zero all of it, load as zeros
    i32x4 x_rows = buffer(qx, rows_x * row_bytes), w_rows = buffer(qw, rows_w * w_row_bytes);
    if constexpr (GATHER) x_rows[2] = __builtin_amdgcn_readfirstlane((int)(uint32_t)min((unsigned long)(p.x_rows - x_first) * (unsigned long)row_bytes, (unsigned long)kGatherMost));
    auto sized = [](i32x4 b, bool live) { return i32x4{b[0], b[1], live ? b[2] : 0, b[3]}; };
    // load i of step kb into the part of LDS at `stage`, the scales last (those of one step after another).  Past the end of K zeros, so
    // that the count of a wave's loads stays the same.
    auto load = [&](int stage, int kb, int i) {
        const bool live = kb < kb1;
        const uint32_t to = lds_at + (uint32_t)stage;
        if (BY == kRowsByExpert && (i == 0 || i == A_LOADS || i >= LOADS) && kb == p.KB - turn) {  // back to the first block
            if (i == 0) {
#pragma unroll
                for (uint32_t &from : x_from) from -= (uint32_t)row_bytes;
            }
            if (i == A_LOADS) w_at -= (uint32_t)w_row_bytes;
            if (i >= LOADS) {
                Scales &of = i == LOADS ? scales : more_scales;
                of.at -= (long)p.KB * of.step;
            }
        }
        if (i < A_LOADS) {
            to_lds16(sized(x_rows, live), to + (uint32_t)(first_x + i * 8 * WN) * kBlock8,
                     GATHER ? x_from[GATHER ? i : 0] + (uint32_t)(kb * kBlock8) : x_at + (uint32_t)(i * 8 * WN * row_bytes + kb * kBlock8));
        } else if (i < LOADS) {
            to_lds16(sized(w_rows, live), to + (uint32_t)(BM * kBlock8 / kWBlock + first_w + (i - A_LOADS) * W_ROWS * W_WAVES) * kWBlock,
                     w_at + (uint32_t)((i - A_LOADS) * W_ROWS * W_WAVES * w_row_bytes + kb * kWBlock));
        } else {
            Scales &of = i == LOADS ? scales : more_scales;
            const uint32_t at = to + (uint32_t)(NUMBERS + (i - LOADS) * 4 * BM + wave * 256);
            const bool words = WBITS == 4 && (WAVES == 8 ? i > LOADS : !scale_x);
            if (words) to_lds4(buffer(of.at, live ? of.rows : 0), at, of.offset);
            else to_lds1(buffer(of.at, live ? of.rows : 0), at, of.offset);
            of.at += of.step;
        }
    };

    f32x4 acc[TM][TN];
#pragma unroll
    for (int i = 0; i < TM; i++)
#pragma unroll
        for (int j = 0; j < TN; j++) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};

    // pieces `quarter` and `quarter` + 4 of a row; products in bf16 by weights of 4 bits take the quarter-th pair
    constexpr bool PAIRS = EXACT && WBITS == 4;
    const int at0 = ((PAIRS ? 2 * quarter : quarter) ^ (l16 & 7)) * 16, at1 = at0 ^ (PAIRS ? 16 : 64);
    const int a_at = (wm * 16 * TM + l16) * kBlock8, b_at = (BM * kBlock8 / kWBlock + wn * 16 * TN + l16) * kWBlock;
    const int at4 = (quarter ^ (l16 >> 2)) * 16;
    auto fragment = [&](const uint8_t *from, int group) {
        const i32x4 low = *reinterpret_cast<const i32x4 *>(from + group * 16 * kBlock8 + at0), high = *reinterpret_cast<const i32x4 *>(from + group * 16 * kBlock8 + at1);
        return (i32x8)__builtin_shufflevector(low, high, 0, 1, 2, 3, 4, 5, 6, 7);
    };
    auto w_fragment = [&](const uint8_t *from, int group) {
        if constexpr (WBITS == 8) return fragment(from, group);
        const i32x4 all = *reinterpret_cast<const i32x4 *>(from + group * 16 * kWBlock + at4);
        return (i32x8)__builtin_shufflevector(all, all, 0, 1, 2, 3, -1, -1, -1, -1);  // (four words are read)
    };
    struct Operands {  // a wave's part of a step
        i32x8 wq[TN], xq[TM];
        ScaleWords<TN> sw;
        ScaleWords<TM> sx;
    };
    constexpr int READS = 1 + TN + TM;
    auto read = [&](Operands &o, int stage, int i) {  // read i of a step
        const uint8_t *const from = lds + stage;
        if (i == 0) {
            const uint32_t *const s_lds = reinterpret_cast<const uint32_t *>(from + NUMBERS);
            o.sw = scale_words<TN>(s_lds + BM + (wn * 16 + l16) * TN);
            if constexpr (WBITS == 4) {
#pragma unroll
                for (int j = 0; j < TN; j++) o.sw.w[j] = o.sw.w[j] >> 8 * quarter & 0xffu;
            }
            o.sx = scale_words<TM>(s_lds + (wm * 16 + l16) * TM);
        } else if (i <= TN) {
            o.wq[i - 1] = w_fragment(from + b_at, i - 1);
        } else {
            o.xq[i - 1 - TN] = fragment(from + a_at, i - 1 - TN);
        }
    };
    auto read_all = [&](Operands &o, int stage) {
#pragma unroll
        for (int i = 0; i < READS; i++) read(o, stage, i);
    };
    // behind each of the first `count` products what `behind` does
    auto multiply = [&](const Operands &o, int count, auto behind) {
        Exact32 wf[EXACT ? TN : 1];
        if constexpr (EXACT) {
#pragma unroll
            for (int j = 0; j < TN; j++) wf[j] = WBITS == 4 ? exact32_of4(o.wq[j], o.sw.w[j]) : exact32<0>(o.wq[j], o.sw.w[j]);
        }
#pragma unroll
        for (int i = 0; i < TM; i++) {
            Exact32 xf;
            if constexpr (EXACT) xf = exact32<FORMAT>(o.xq[i], o.sx.w[i]);
#pragma unroll
            for (int j = 0; j < TN; j++) {
                if constexpr (EXACT) acc[i][j] = mfma16_exact(wf[j], xf, acc[i][j]);
                else acc[i][j] = mfma16<FORMAT, WBITS>(o.wq[j], o.xq[i], acc[i][j], o.sw.w[j], o.sx.w[i]);
                if (i * TN + j < count) {
                    behind(i * TN + j);
                    __builtin_amdgcn_sched_barrier(0);
                }
            }
            __builtin_amdgcn_sched_barrier(0);
        }
#pragma unroll
        for (int l = TM * TN; l < count; l++) behind(l);
    };
    auto barrier = [] {
        asm volatile("" ::: "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
    };
    auto all_read = [] { __builtin_amdgcn_s_waitcnt(0xc07f); };  // this wave's reads of LDS are done
    auto load_first = [&] {
#pragma unroll
        for (int k = 0; k < STAGES; k++)
#pragma unroll
            for (int i = 0; i <= LOADS; i++) load(k * STAGE, kb0 + k, i);
    };
    if constexpr (WAVES == 8) {
        // Two waves a SIMD take turns: while one multiplies the other reads, a barrier at every change.  Slot 2s: the first four waves read step s, the
        // others multiply step s - 1; slot 2s + 1 the other way round.  Of a step's part of LDS the rows of X that only the first four waves
        // read are free from slot 2s + 1 on, where those load theirs of step s + 2; the rest from slot 2s + 2 on, the slot in which the first four
        // waves load W and the scales of step s + 2 (which slot 2s + 4 reads), and 2s + 3, in which the others load their rows of X (for slot 2s + 5).
        // Few loads go out between the products: a wave that waits to get one out does not multiply.
        static_assert(STAGES == 2, "two steps in LDS");
        // (An expert's last tile is rarely full: with at most half the rows the second four waves have nothing to multiply.  Leaving groups of 16 rows out one by
        // one instead cost full tiles 3-5 %.)
        constexpr bool HALF = BY == kRowsByExpert;
        Operands o;
        if (wm == 0) {
#pragma unroll
            for (int i = 0; i < LOADS + 2; i++) load(0, kb0, i);
#pragma unroll
            for (int i = 0; i < A_LOADS; i++) load(STAGE, kb0 + 1, i);
            wait_loads<A_LOADS>();
            barrier();
            for (int kb = kb0; kb < kb1; kb++) {
                const int stage = (kb - kb0) & 1 ? STAGE : 0;
                read_all(o, stage);
#pragma unroll
                for (int i = A_LOADS; i < LOADS + 2; i++) load(STAGE - stage, kb + 1, i);
                all_read();
                barrier();
                __builtin_amdgcn_s_setprio(1);
                multiply(o, TM * TN, [&](int i) {
                    if (i % (TM * TN / A_LOADS) == 0) load(stage, kb + 2, i / (TM * TN / A_LOADS));
                });
                __builtin_amdgcn_s_setprio(0);
                wait_loads<A_LOADS>();
                barrier();
            }
            barrier();
        } else {
#pragma unroll
            for (int i = 0; i < A_LOADS; i++) load(0, kb0, i);
            wait_loads<0>();
            barrier();
            barrier();
            for (int kb = kb0; kb < kb1; kb++) {
                const int stage = (kb - kb0) & 1 ? STAGE : 0;
                read_all(o, stage);
#pragma unroll
                for (int i = 0; i < A_LOADS; i++) load(STAGE - stage, kb + 1, i);
                all_read();
                barrier();
                __builtin_amdgcn_s_setprio(1);
                if (!HALF || rows_x > BM / 2) multiply(o, 0, [](int) {});
                __builtin_amdgcn_s_setprio(0);
                wait_loads<0>();
                barrier();
            }
        }
    } else if constexpr (EXACT && BM * BN > 64 * 128) {
        // no registers for two steps' operands
        static_assert(STAGES == 2, "steps in LDS");
        load_first();
        Operands o;
        for (int kb = kb0, stage = 0; kb < kb1; kb++, stage = STAGE - stage) {
            wait_loads<LOADS + 1>();  // this wave's part of the step has landed,
            barrier();                // and so has the others'
            read_all(o, stage);
            all_read();
            barrier();                // the step's part of LDS is free
            multiply(o, LOADS + 1, [&](int i) { load(stage, kb + 2, i); });
        }
    } else {
        // a step's operands are read from LDS while the step before is multiplied
        Operands even, odd;
        auto step = [&](const Operands &now, Operands &next, int kb, int stage) {
            wait_loads<(STAGES - 2) * (LOADS + 1)>();  // this wave's part of the next step has landed,
            all_read();                                // it has read all of this one,
            barrier();                                 // and so have the others: this one's part of LDS is free
            multiply(now, READS > LOADS + 1 ? READS : LOADS + 1, [&](int i) {
                if (i < READS) read(next, stage == (STAGES - 1) * STAGE ? 0 : stage + STAGE, i);
                if (i <= LOADS) load(stage, kb + STAGES, i);
            });
        };
        load_first();
        wait_loads<(STAGES - 1) * (LOADS + 1)>();
        barrier();
        read_all(even, 0);
        if constexpr (STAGES == 3) {  // places in LDS are constants of the code
            for (int kb = kb0; BY == kOneWeight || kb < kb1; kb += 6) {  // (an expert may have no steps)
                step(even, odd, kb, 0);
                if (kb + 1 >= kb1) break;
                step(odd, even, kb + 1, STAGE);
                if (kb + 2 >= kb1) break;
                step(even, odd, kb + 2, 2 * STAGE);
                if (kb + 3 >= kb1) break;
                step(odd, even, kb + 3, 0);
                if (kb + 4 >= kb1) break;
                step(even, odd, kb + 4, STAGE);
                if (kb + 5 >= kb1) break;
                step(odd, even, kb + 5, 2 * STAGE);
                if (kb + 6 >= kb1) break;
            }
        } else {  // (with constants the largest of these tiles needs more registers than there are)
            static_assert(STAGES == 2, "steps in LDS");
            int stage = 0;
            for (int kb = kb0; kb < kb1; kb += 2) {
                step(even, odd, kb, stage);
                stage = stage == STAGE ? 0 : STAGE;
                if (kb + 1 < kb1) {
                    step(odd, even, kb + 1, stage);
                    stage = stage == STAGE ? 0 : STAGE;
                }
            }
        }
    }
    wait_loads<0>();  // nothing is on its way to LDS any more,
    __builtin_amdgcn_s_barrier();  // and every wave has read its last step: LDS is free
    asm volatile("" ::: "memory");

    // The weights are the instruction's rows: a lane holds four neighbours of one row of Y.  Rows of 16 at a time go through a part of LDS of the
    // wave's own, so that they are stored in pieces of 16 bytes and whole cache lines (four neighbours a lane, straight from the registers:
    // 25 us for a tile of 256 x 256, a fifth of 8192^3).
    constexpr int V = 16 / (int)sizeof(T), PIECES = TN * 16 / V, PITCH = TN * 16 * (int)sizeof(T) + 16;
    static_assert(WAVES * 16 * PITCH <= STAGES * STAGE, "the waves' parts fit");
    uint8_t *const mine = lds + wave * (16 * PITCH);
    T *const y = static_cast<T *>(p.y) + (long)(BY == kKByExpert ? expert : part) * p.M * p.N;
    struct __attribute__((packed, aligned(sizeof(T)))) Piece { T v[V]; };
    struct alignas(4 * sizeof(T)) Four { T v[4]; };
#pragma unroll
    for (int i = 0; i < TM; i++) {
#pragma unroll
        for (int j = 0; j < TN; j++)
            *reinterpret_cast<Four *>(mine + l16 * PITCH + (j * 16 + quarter * 4) * (int)sizeof(T)) =
                Four{{(T)acc[i][j][0], (T)acc[i][j][1], (T)acc[i][j][2], (T)acc[i][j][3]}};
#pragma unroll
        for (int c = 0; c < 16 * PIECES / 64; c++) {
            const int piece = c * 64 + lane, row = piece / PIECES, column = piece % PIECES * V;
            const Piece v = *reinterpret_cast<const Piece *>(mine + row * PITCH + column * (int)sizeof(T));
            const int m = m0 + (wm * TM + i) * 16 + row, n = n0 + wn * TN * 16 + column;
            if (m >= end_m) continue;
            T *const to = y + (long)m * p.N + n;
            if (p.streamed) {  // (rows are whole cache lines)
                typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
                if (n < p.N) __builtin_nontemporal_store(__builtin_bit_cast(u32x4, v), reinterpret_cast<u32x4 *>(to));
            } else if (n + V <= p.N) {
                *reinterpret_cast<Piece *>(to) = v;
            } else {
#pragma unroll
                for (int e = 0; e < V; e++)
                    if (n + e < p.N) to[e] = v.v[e];
            }
        }
    }
}

// The parts of a K that was split over workgroups, added up in their order and rounded once (so the same call gives the same bits, which sums by
// atomics would not).  Memory bound, and a launch: about 2.5 us for 4 parts of 64 x 4096.
template <int OUT> __global__ __launch_bounds__(256) void linear8_join(const float *parts, void *y, long count, int n)
{
    using T = typename Element<OUT>::type;
    const long i = ((long)blockIdx.x * 256 + threadIdx.x) * 4;
    if (i >= count) return;
    if (count % 4 == 0) {
        f32x4 sum = *reinterpret_cast<const f32x4 *>(parts + i);
        for (int k = 1; k < n; k++) sum += *reinterpret_cast<const f32x4 *>(parts + k * count + i);
        store4(static_cast<T *>(y) + i, sum);
    } else {
        for (long j = i; j < min(i + 4, count); j++) {
            float sum = parts[j];
            for (int k = 1; k < n; k++) sum += parts[k * count + j];
            static_cast<T *>(y)[j] = (T)sum;
        }
    }
}

// Few rows: bound by reading QW once.  A workgroup takes some groups of 16 rows of QW and all rows of X, or a part of them (at most 16 * MT).  Its waves take the blocks of
// K in turn, each lane loads its 2 x 16 bytes of a block of QW itself, AHEAD blocks at a time, and the waves' sums meet in LDS, added up in a
// fixed order.  X lies in LDS as packed numbers (rows 16 bytes more than whole blocks apart, so that 8 rows' pieces meet different banks) and scales:
// INPUT 0 .. 2: fp32 / bf16 / fp16, quantized by the workgroup on the way (a block of a row is 16 lanes of eight); 3: packed.
// One row of 4096 by 4096 x 4096: 4.6-6.0 us with its launch, 16.9 MB at 2.8-3.6 TB/s (through the tiles and a launch of the quantizer 14); of 4 bits 4.2, 8.9 MB,
// most of it the launch.  24 rows of 2050 (fp16) by 1003: 5.4 us, of 4 bits 4.6, bound by every workgroup's conversion of its rows of X (of all of them 9.3-10.4),
// which costs less than a launch for it alone; 16 waves instead of 8 took 5.9-6.4 and (of all rows) 10.9-11.2 us.
struct RowsParams {
    const void *x;
    const uint8_t *sx, *qw, *sw;
    void *y;
    int M, N, K, KB, w_scale_rows, groups_each, rows_each;  // rows_each: of X, of a workgroup
    long ldx;
    Div32 div_kb;
};

// The bound between one launch and quantizer, tiles and join: X in 72 KB of LDS, which up to 16 rows (with 8 KB for the waves' sums) leaves room for two workgroups
// a CU; with 17 to 32 rows the sums take 16 KB, and a CU holds one.  On both sides of it (bf16, by 4096 columns, a pass among others, us):
//   one launch   8 x 4096  7.6   12 x 4096  9.2   17 x 4096 11.9   8 x 8000 15.0   32 x 2176  9.7   32 x 1000 7.0   by 1003 columns 24 x 2050 5.4, 32 x 2050 5.7
//   three        18 x 4096 10.0                                    8 x 9300 12.7   32 x 2304  8.6   33 x 1000 7.4   by 1003 columns 33 x 2050 8.8
// So the largest X in one launch take up to a fifth longer than three launches would; they meet at about 12 rows of 4096.
constexpr int kRowsMost = 32;           // rows of X
constexpr int kRowsLds = 72 << 10;      // bytes of X in LDS
constexpr int kRowsWaves = 8;

__host__ __device__ __forceinline__ int rows_stride(int KB) { return KB * kBlock8 + 16; }
__host__ __device__ __forceinline__ int rows_lds(int M, int KB) { return M * (rows_stride(KB) + KB * 4); }  // numbers, then scales as words [KB][M]

// A lane's part of a block of W
template <int WBITS> __device__ __forceinline__ i32x8 w_numbers(i32x4 low, i32x4 high)
{
    if constexpr (WBITS == 8) return __builtin_shufflevector(low, high, 0, 1, 2, 3, 4, 5, 6, 7);
    else return __builtin_shufflevector(low, low, 0, 1, 2, 3, -1, -1, -1, -1);
}

// 16 rows of W by 16 rows of X in LDS, one block of K: x is the lane's row's block.  (Which numbers a lane takes: as in the tiles.)
template <int FORMAT, int OUT, int WBITS> __device__ __forceinline__ f32x4 times_rows(i32x8 w, uint32_t w_scale, const uint8_t *x, uint32_t x_scale, int quarter, f32x4 c)
{
    constexpr bool PAIRS = OUT == 0 && WBITS == 4;
    x += quarter * (PAIRS ? 32 : 16);
    const i32x4 low = *reinterpret_cast<const i32x4 *>(x), high = *reinterpret_cast<const i32x4 *>(x + (PAIRS ? 16 : 64));
    const i32x8 xf = __builtin_shufflevector(low, high, 0, 1, 2, 3, 4, 5, 6, 7);
    if constexpr (OUT == 0) return mfma16_exact(WBITS == 4 ? exact32_of4(w, w_scale) : exact32<0>(w, w_scale), exact32<FORMAT>(xf, x_scale), c);
    else return mfma16<FORMAT, WBITS>(w, xf, c, w_scale, x_scale);
}

template <int INPUT, int FORMAT, int OUT, int MT, int WBITS = 8>
__global__ __launch_bounds__(64 * kRowsWaves) void linear8_rows(const RowsParams p)
{
    using T = typename Element<OUT>::type;
    constexpr int WAVES = kRowsWaves, AHEAD = 4, kWBlock = kBlock8 * WBITS / 8;
    extern __shared__ __attribute__((aligned(16))) uint8_t packed[];
    __shared__ __attribute__((aligned(16))) float sums[WAVES * MT * 256];
    const int t = threadIdx.x, lane = t % 64, wave = __builtin_amdgcn_readfirstlane(t / 64), l16 = lane % 16, quarter = lane / 16;
    const int stride = rows_stride(p.KB), m0 = (int)blockIdx.y * p.rows_each, M = min(p.rows_each, p.M - m0);
    uint32_t *const scales = reinterpret_cast<uint32_t *>(packed + M * stride);
    const bool w_rows = p.w_scale_rows == p.N;
    // block u of the AHEAD that a wave takes from `first` on: every eighth one, or (of 4 bits) every eighth pair, which is a cache line
    auto block_of = [](int first, int u) { return WBITS == 4 ? first + u / 2 * (2 * WAVES) + u % 2 : first + u * WAVES; };
    const int wave_first = WBITS == 4 ? 2 * wave : wave;
    i32x4 w_low[AHEAD], w_high[WBITS == 8 ? AHEAD : 1];
    uint32_t w_scale[AHEAD];
    auto load = [&](int n0, int first) {
        const int row = min(n0 + l16, p.N - 1);
        const uint8_t *const w = p.qw + (long)row * p.KB * kWBlock + quarter * 16, *const s = WBITS == 4 ? p.sw + row * 4 + quarter : p.sw + (w_rows ? row : row / kBlock8);
#pragma unroll
        for (int u = 0; u < AHEAD; u++) {
            const long kb = min(block_of(first, u), p.KB - 1);
            w_low[u] = *reinterpret_cast<const i32x4 *>(w + kb * kWBlock);
            if constexpr (WBITS == 8) w_high[u] = *reinterpret_cast<const i32x4 *>(w + kb * kWBlock + 64);
            w_scale[u] = s[kb * p.w_scale_rows * (WBITS == 4 ? 4 : 1)];
        }
    };
    const int groups = (p.N + 15) / 16, group0 = (int)blockIdx.x * p.groups_each, group1 = min(groups, group0 + p.groups_each);
    load(group0 * 16, wave_first);

    // X into LDS: blocks in the order of memory, 16 lanes a block, AT_ONCE of them on their way
    constexpr int AT_ONCE = 8, STEP = 64 * WAVES / 16;
    const int blocks = M * p.KB;
    for (int first = t / 16; first < blocks; first += AT_ONCE * STEP) {
        using X = typename Element<INPUT == 3 ? 0 : INPUT>::type;
        Words<X> v[AT_ONCE];
#pragma unroll
        for (int u = 0; u < AT_ONCE; u++) {
            const int block = first + u * STEP, m = (int)div32(block, p.div_kb), kb = block - m * p.KB;
            if (block >= blocks) break;
            if constexpr (INPUT == 3) {
                const uint2 w = *reinterpret_cast<const uint2 *>(static_cast<const uint8_t *>(p.x) + ((long)m0 * p.KB + block) * kBlock8 + l16 * 8);
                v[u].w[0] = w.x, v[u].w[1] = w.y, v[u].w[2] = p.sx[(long)kb * p.M + m0 + m];
            } else {
                v[u] = load_words(static_cast<const X *>(p.x) + (m0 + m) * p.ldx, kb * kBlock8 + l16 * 8, p.K);
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
            if (l16 == 0) scales[kb * M + m] = byte;
        }
    }
    __syncthreads();

    for (int group = group0; group < group1; group++) {
        const int n0 = group * 16;
        f32x4 acc[MT];
#pragma unroll
        for (int i = 0; i < MT; i++) acc[i] = f32x4{0.f, 0.f, 0.f, 0.f};
        for (int first = wave_first; first < p.KB; first += AHEAD * WAVES) {
            if (first != wave_first) load(n0, first);
#pragma unroll
            for (int u = 0; u < AHEAD; u++) {
                const int kb = block_of(first, u);
                if (kb >= p.KB) break;  // (the same for the whole wave)
                const i32x8 wf = w_numbers<WBITS>(w_low[u], w_high[WBITS == 8 ? u : 0]);
#pragma unroll
                for (int i = 0; i < MT; i++) {
                    const int m = min(i * 16 + l16, M - 1);  // (columns past M repeat the last one and are not stored)
                    acc[i] = times_rows<FORMAT, OUT, WBITS>(wf, w_scale[u], packed + m * stride + kb * kBlock8, scales[kb * M + m], quarter, acc[i]);
                }
            }
        }
        if (group + 1 < group1) load(n0 + 16, wave_first);  // the next group's first blocks, on their way while the sums meet
#pragma unroll
        for (int i = 0; i < MT; i++) *reinterpret_cast<f32x4 *>(sums + (wave * MT + i) * 256 + l16 * 16 + quarter * 4) = acc[i];
        __syncthreads();
        for (int i = t; i < MT * 256; i += 64 * WAVES) {
            const int m = i / 16, n = n0 + i % 16;
            float sum = sums[i];
#pragma unroll
            for (int k = 1; k < WAVES; k++) sum += sums[k * MT * 256 + i];
            if (m < M && n < p.N) static_cast<T *>(p.y)[(long)(m0 + m) * p.N + n] = (T)sum;
        }
        if (group + 1 < group1) __syncthreads();
    }
}

// The rows of X are cut up among workgroups while a CU gets one at the most: each converts its own rows alone.  Whole / cut, in a replayed graph, 4 bits, bf16, us:
// by 1003 columns (four cuts) 24 x 2050 7.9 / 4.5, 16 x 4096 8.3 / 4.8; by 2048 (two) 16 x 4096 8.2 / 6.0; by 4096, where two cuts would be two workgroups a CU,
// 8.4 / 8.5; more than 16 cuts gain nothing (128 x 4096 by 64: eight 8.3, sixteen 5.9).
inline int rows_cuts(int M, int groups)
{
    const int free = groups < 256 ? 256 / groups : 1, cuts = free < 16 ? free : 16;
    return cuts < M ? cuts : M;
}

// One launch, where a workgroup's rows of X fit.  With weights of 4 bits that goes by the rows after the cut: one launch / three, bf16, us: by 64 columns 128 x 4096
// 5.9 / 11.5, 256 x 1024 5.0 / 7.7; by 1003 64 x 4096 8.6 / 10.4, 32 x 8192 11.9 / 12.3; by 2048 64 x 2050 9.5 / 9.3.  With weights of 8 bits by all rows,
// as before the cut: the ways differ in the order of their sums, and a product keeps its bits.
inline bool rows_fit(int M, int KB) { return M <= kRowsMost && KB <= kRowsLds / kBlock8 && rows_lds(M, KB) <= kRowsLds; }
template <int WBITS> bool rows_way(int M, int N, int KB)
{
    if (WBITS == 8) return rows_fit(M, KB);
    const int cuts = rows_cuts(M, (N + 15) / 16);
    return rows_fit((M + cuts - 1) / cuts, KB);
}

template <int INPUT, int FORMAT, int OUT, int WBITS = 8> hipError_t launch_rows(RowsParams p, hipStream_t stream)
{
    const int groups = (p.N + 15) / 16;
    p.groups_each = (groups + 511) / 512;  // two workgroups a CU, each with X in its LDS once
    const int cuts = rows_cuts(p.M, groups);
    p.rows_each = (p.M + cuts - 1) / cuts;
    const dim3 workgroups((unsigned)((groups + p.groups_each - 1) / p.groups_each), (unsigned)((p.M + p.rows_each - 1) / p.rows_each));
    const unsigned lds = (unsigned)rows_lds(p.rows_each, p.KB);
    if (p.rows_each <= 16) linear8_rows<INPUT, FORMAT, OUT, 1, WBITS><<<workgroups, 64 * kRowsWaves, lds, stream>>>(p);
    else linear8_rows<INPUT, FORMAT, OUT, 2, WBITS><<<workgroups, 64 * kRowsWaves, lds, stream>>>(p);
    return hipGetLastError();
}

inline int w_scale_rows(int N, int w_block_rows) { return w_block_rows == 1 ? N : (N + kBlock8 - 1) / kBlock8; }

struct Plan8 {
    int rows, columns;  // of the tile
    int parts, kb_per_part;
    long tiles;
};

// The tile and the parts that K is cut into: the least of what a launch takes by the busiest CU's work.  A step of one of the tiles that a CU holds at
// once takes `alone` us (latency) or, of all its tiles, `among` (throughput), a tile's way out `out`; parts are written in fp32, read and added
// up by a launch of their own.  Constants fitted to every (tile, parts) of 60 products of 33 .. 16384 rows, 64 .. 8192 columns and K on an MI355X, with weights of 8
// bits and before outputs left past the caches; what they pick now, over the best, on 132 other products, mean and worst:
//   8 bits   500 and more rows 1.2 %, 13 % (5423 x 394 over 538)   34 .. 550 rows 4.3 %, 53 % (99 x 78 over 7912)   fp32 1.4 %, 12 % (2749 x 468 over 133)
//   4 bits                     2.9 %, 24 % (the same)                             2.4 %, 16 %                            1.8 %, 11 %
struct TileTimes { int rows, columns, held; double alone, among, out; };
// The same of tiles over experts (16-bit sums, and full ones); their ways out are shorter, past the caches
constexpr TileTimes kExpertTiles[] = {{64, 64, 3, 0.092, 0.165, 0.46}, {64, 128, 2, 0.237, 0.235, 0.725}, {128, 128, 2, 0.509, 0.41, 0.923}, {256, 256, 1, 0.96, 0.945, 2.854}};
constexpr TileTimes kExpertExact[] = {{64, 64, 3, 0.371, 0.242, 0.7}, {64, 128, 2, 0.553, 0.336, 1.32}, {128, 128, 2, 1.22, 0.716, 1.65}};

inline Plan8 plan8(int out, int M, int N, int KB)
{
    constexpr TileTimes kFast[] = {{64, 64, 3, 0.05, 0.174, 0.8}, {64, 128, 2, 0.171, 0.242, 1.37}, {128, 128, 2, 0.571, 0.473, 1.69}, {256, 256, 1, 1.235, 1.125, 6.25}};
    constexpr TileTimes kExact[] = {{64, 64, 3, 0.371, 0.242, 0.7}, {64, 128, 2, 0.553, 0.336, 1.32}, {128, 128, 2, 1.22, 0.716, 1.65}};
    const double join = out == 0 ? 2.5 : 1.9, join_part = out == 0 ? 0.936e-6 : 0.747e-6, join_out = out == 0 ? 0.008e-6 : 0;
    Plan8 best = {};
    double least = 1e30;
    for (int i = 0; i < (out == 0 ? 3 : 4); i++) {
        const TileTimes &tile = out == 0 ? kExact[i] : kFast[i];
        const long tiles = ((M + (long)tile.rows - 1) / tile.rows) * ((N + (long)tile.columns - 1) / tile.columns);
        for (int parts = 1; parts <= 16 && parts <= KB; parts *= 2) {
            if (parts > 1 && tiles * parts > 2048) break;
            const int steps = (KB + parts - 1) / parts;
            if ((KB + steps - 1) / steps != parts) continue;
            const long each = (tiles * parts + 255) / 256, rounds = (each + tile.held - 1) / tile.held;
            const double alone = tile.alone * (double)rounds, among = tile.among * (double)each;
            double t = steps * (alone > among ? alone : among) + tile.out * (double)each * (parts > 1 || out == 0 ? 2 : 1);
            if (parts > 1) t += join + (parts * join_part + join_out) * (double)M * (double)N;
            if (t < least) {
                least = t;
                best = {tile.rows, tile.columns, parts, steps, tiles};
            }
        }
    }
    return best;
}

// Whether Y (`count` elements of type `out` in rows of N) is written past the caches: from 16 MB on, where its rows are whole cache lines, which a wave then
// writes at once.  What is smaller is read from the caches by the next kernel.  16384 x 2048 bf16, two tiles a CU: the way out 21 -> 11 us.  With the quantizer
// that reads Y behind it, in a replayed graph, us through / past the caches: 1024 x 4096 over 4096 27.5 / 27.3, 2048 x 2048 over 2048 19.4 / 19.2, 4096 x 2048 over 4096
// 40.2 / 39.1, 4096 x 4096 over 2048 40.9 / 41.5, 8192 x 8192 over 8192 423 / 415.
inline int streamed(int out, const void *y, long count, int N)
{
    const long bytes = out == 0 ? 4 : 2;
    return count * bytes >= 16l << 20 && (N * bytes) % 128 == 0 && (uintptr_t)y % 128 == 0;
}

inline int threads_of(const Plan8 &plan) { return plan.rows == 256 ? 512 : 256; }

template <int FORMAT, int OUT, bool EXACT, int WBITS = 8, int BY = kOneWeight>
hipError_t launch_tiles(const Plan8 &plan, long groups, const typename TileParamsOf<BY>::type &p, hipStream_t stream)
{
    const unsigned n = (unsigned)groups;
    if constexpr (!EXACT)
        if (plan.rows == 256) {
            linear8_tiles<256, 256, 2, 4, 2, FORMAT, OUT, EXACT, WBITS, BY><<<n, threads_of(plan), 0, stream>>>(p);
            return hipGetLastError();
        }
    if (plan.rows == 128) linear8_tiles<128, 128, 2, 2, 2, FORMAT, OUT, EXACT, WBITS, BY><<<n, threads_of(plan), 0, stream>>>(p);
    else if (plan.columns == 128) linear8_tiles<64, 128, 2, 2, 3, FORMAT, OUT, EXACT, WBITS, BY><<<n, threads_of(plan), 0, stream>>>(p);
    else linear8_tiles<64, 64, 2, 2, 3, FORMAT, OUT, EXACT, WBITS, BY><<<n, threads_of(plan), 0, stream>>>(p);
    return hipGetLastError();
}

// Y from its parts
inline hipError_t launch_join(int out, const float *parts, void *y, long count, int n, hipStream_t stream)
{
    const unsigned joins = (unsigned)((count + 1023) / 1024);
    if (out == 0) linear8_join<0><<<joins, 256, 0, stream>>>(parts, y, count, n);
    else if (out == 1) linear8_join<1><<<joins, 256, 0, stream>>>(parts, y, count, n);
    else linear8_join<2><<<joins, 256, 0, stream>>>(parts, y, count, n);
    return hipGetLastError();
}

// One product of a packed activation: few rows, or tiles, with a launch that joins the parts of K
template <int FORMAT, int WBITS> hipError_t launch_product(int out, const Linear8Args &a, int scale_rows, void *workspace, hipStream_t stream)
{
    if (rows_way<WBITS>(a.M, a.N, a.KB)) {
        const RowsParams p = {a.qx, a.sx, a.qw, a.sw, a.y, a.M, a.N, a.KB * kBlock8, a.KB, scale_rows, 0, 0, 0, make_div32((uint32_t)a.KB)};
        return out == 0 ? launch_rows<3, FORMAT, 0, WBITS>(p, stream) : out == 1 ? launch_rows<3, FORMAT, 1, WBITS>(p, stream) : launch_rows<3, FORMAT, 2, WBITS>(p, stream);
    }
    const Plan8 plan = plan8(out, a.M, a.N, a.KB);
    const int tiles_m = (a.M + plan.rows - 1) / plan.rows, tiles_n = (a.N + plan.columns - 1) / plan.columns;
    const TileParams p = {a.qx, a.sx, a.qw, a.sw, plan.parts > 1 ? workspace : a.y, a.M, a.N, a.KB, scale_rows, plan.kb_per_part, tiles_m, tiles_n,
                          plan.parts == 1 && plan.rows * plan.columns > 64 * 64 && streamed(out, a.y, (long)a.M * a.N, a.N)};
    const long groups = plan.tiles * plan.parts;
    if (plan.parts == 1)
        return out == 0 ? launch_tiles<FORMAT, 0, true, WBITS>(plan, groups, p, stream)
                        : out == 1 ? launch_tiles<FORMAT, 1, false, WBITS>(plan, groups, p, stream) : launch_tiles<FORMAT, 2, false, WBITS>(plan, groups, p, stream);
    const hipError_t e = out == 0 ? launch_tiles<FORMAT, 0, true, WBITS>(plan, groups, p, stream) : launch_tiles<FORMAT, 0, false, WBITS>(plan, groups, p, stream);
    return e != hipSuccess ? e : launch_join(out, static_cast<const float *>(workspace), a.y, (long)a.M * a.N, plan.parts, stream);
}

}  // namespace

}  // namespace tab
