// Product of two packed 8-bit operands with power-of-two scales per block of 128,
//   Y[m][n] = sum over kb of 2^(SX[kb][m] + SW[kb][n] - 254) * sum over k in block kb of QX[m][k] QW[n][k].
//
// 16-bit outputs: v_mfma_scale_f32_16x16x128_f8f6f4.  One instruction is a 16 x 16 tile over one block of K, and it takes the E8M0 bytes of its
// 16 rows and 16 columns as operands, so the scales cost no vector instruction and the sums stay in one set of fp32 accumulators.  Inside
// the instruction, products of eight neighbours in K are aligned to the largest of them and keep 13 bits below it (measured): 1.5e-5 of the
// output's size for normal operands, far below the 2^-8 or 2^-11 of the output's own rounding, but not what an fp32 output is for.  (512 x 4096 x 4096: 1.2 % of
// the bf16 outputs are the other neighbour of what the fp32 output rounds to; off the fp32 output by 0.0016633 of its size instead of 0.0016632.)
// fp32 outputs (EXACT): the numbers times their scales are bf16 numbers exactly (4 of 8 significant bits, the exponent range of fp32), made by one
// conversion of two numbers, and v_mfma_f32_16x16x32_bf16 multiplies them at half the rate with full fp32 sums.  A number below 2^-126 may
// count as zero there.
#include "tab_blocks8.h"
#include "tab_common.h"

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
};

template <int FORMAT> __device__ __forceinline__ f32x4 mfma16(i32x8 w, i32x8 x, f32x4 c, uint32_t w_scale, uint32_t x_scale)
{
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(w, x, c, 0, FORMAT, 0, (int)w_scale, 0, (int)x_scale);
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
__device__ __forceinline__ uint32_t lds_address(const uint8_t *p) { return (uint32_t)(uintptr_t)(const __attribute__((address_space(3))) uint8_t *)p; }

// A buffer of `bytes` (below 2^31; none if negative) from p on, the same in every lane: base, size, flags
__device__ __forceinline__ i32x4 buffer(const uint8_t *p, int bytes)
{
    const uint64_t at = (uint64_t)p;
    return i32x4{__builtin_amdgcn_readfirstlane((int)(uint32_t)at), __builtin_amdgcn_readfirstlane((int)(at >> 32) & 0xffff),
                 __builtin_amdgcn_readfirstlane(max(bytes, 0)), kBufferFlags8};
}

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
//   256 x 256  8192^3 404-406 us, 2.7 PFLOP/s, in a replayed graph (432-442 with X's quantizer; 430-460 under a profiler's trace; a library's fp8 product with one
//              scale a tensor 361)
//   128 x 128  4096 x 2048 x 4096 37-41 us, 1.7-1.9 PFLOP/s
//   64 x 128   512 x 4096 x 4096 13.8 us, 1.25 PFLOP/s (64 x 64 16.4; both 19 with read and multiplied in turn)
//   64 x 64    128 x 4096 x 4096 9.0 us (14.0 in turn); fp32 1000 x 776 x 520 6.6 us
// A step is one block of K: 128 bytes of each of the tile's rows and their scales,
// straight from global memory into one of STAGES parts of LDS.  A row is eight pieces of 16 bytes; row r has piece g at place g ^ (r & 7), so
// that lanes that read at once meet different banks.  Which piece a lane multiplies is free as long as both operands agree, since a block
// has one scale.
template <int BM, int BN, int WM, int WN, int STAGES, int FORMAT, int OUT, bool EXACT>
__global__ __launch_bounds__(64 * WM * WN, 2) void linear8_tiles(const TileParams p)
{
    using T = typename Element<OUT>::type;
    constexpr int WAVES = WM * WN, THREADS = 64 * WAVES, TM = BM / WM / 16, TN = BN / WN / 16;
    constexpr int NUMBERS = (BM + BN) * kBlock8, STAGE = NUMBERS + 4 * THREADS;
    constexpr int W_WAVES = WAVES == 8 ? WN : WAVES;  // of eight waves the first four load W and the scales
    constexpr int A_LOADS = BM / 8 / WAVES, W_LOADS = BN / 8 / W_WAVES, LOADS = A_LOADS + W_LOADS;
    static_assert(BM + BN <= THREADS, "a lane loads one scale");
    __shared__ __attribute__((aligned(1024))) uint8_t lds[STAGES * STAGE];

    // the tile: parts of K outermost; every XCD (workgroup number modulo 8) takes one run of the tiles, and a run goes through
    // groups of 8 tiles of rows, so that what its CUs hold at one time reads few rows of either operand
    const uint32_t tiles = (uint32_t)p.tiles_m * (uint32_t)p.tiles_n, part = blockIdx.x / tiles, b = blockIdx.x - part * tiles, share = tiles / 8;
    const uint32_t id = b < share * 8 ? (b & 7) * share + (b >> 3) : b;
    const uint32_t in_group = 8 * (uint32_t)p.tiles_n, group = id / in_group, rest = id - group * in_group;
    const uint32_t rows = min(8u, (uint32_t)p.tiles_m - group * 8), tile_n = rest / rows, tile_m = group * 8 + rest - tile_n * rows;
    const int m0 = (int)tile_m * BM, n0 = (int)tile_n * BN;
    const int kb0 = (int)part * p.kb_per_part, kb1 = min(p.KB, kb0 + p.kb_per_part);

    const int t = threadIdx.x, lane = t % 64, wave = __builtin_amdgcn_readfirstlane(t / 64), wm = wave / WN, wn = wave % WN, l16 = lane % 16, quarter = lane / 16;
    const int row_bytes = p.KB * kBlock8, rows_x = min(BM, p.M - m0), rows_w = min(BN, p.N - n0);
    const uint8_t *const qx = p.qx + (long)m0 * row_bytes, *const qw = p.qw + (long)n0 * row_bytes;
    // load i of a wave is eight rows of an operand's tile, eight lanes a row: of W the waves take turns, of X those that multiply the rows
    const int first_x = wm * (BM / WM) + wn * 8, first_w = wave * 8;
    const uint32_t x_at = (uint32_t)(first_x + lane / 8) * (uint32_t)row_bytes + (uint32_t)((lane % 8) ^ (lane / 8)) * 16;
    const uint32_t w_at = (uint32_t)(first_w + lane / 8) * (uint32_t)row_bytes + (uint32_t)((lane % 8) ^ (lane / 8)) * 16;
    // A lane loads one scale: place t of X's, then of W's (of eight waves the first four load one of each).  The scales of a lane's groups of 16 rows are
    // side by side.  (A wave's scales are all of X or all of W.)
    const bool row_scales = p.w_scale_rows == p.N;
    struct Scales { const uint8_t *at; int step, rows; uint32_t offset; };
    auto scales_of = [&](bool x, int place, bool any) {
        const int groups = x ? TM : TN, row = place / (16 * groups) * (16 * groups) + place % groups * 16 + place / groups % 16, step = x ? p.M : p.w_scale_rows;
        return Scales{(x ? p.sx + m0 : p.sw + (row_scales ? n0 : n0 / kBlock8)) + (long)kb0 * step, step,
                      !any ? 0 : x ? rows_x : row_scales ? rows_w : (n0 + rows_w - 1) / kBlock8 - n0 / kBlock8 + 1,
                      (uint32_t)(x || row_scales ? row : (n0 + row) / kBlock8 - n0 / kBlock8)};
    };
    const bool scale_x = WAVES == 8 || wave * 64 < BM;
    Scales scales = scales_of(scale_x, scale_x ? t : t - BM, wave * 64 < BM + BN), more_scales = scales_of(false, t, true);
    const uint32_t lds_at = lds_address(lds);
    // the rows of an operand's tile are one buffer: rows past its end, and with a size of zero all of it, load as zeros
    const i32x4 x_rows = buffer(qx, rows_x * row_bytes), w_rows = buffer(qw, rows_w * row_bytes);
    auto sized = [](i32x4 b, bool live) { return i32x4{b[0], b[1], live ? b[2] : 0, b[3]}; };
    // load i of step kb into the part of LDS at `stage`, the scales last (those of one step after another).  Past the end of K zeros, so
    // that the count of a wave's loads stays the same.
    auto load = [&](int stage, int kb, int i) {
        const bool live = kb < kb1;
        const uint32_t to = lds_at + (uint32_t)stage;
        if (i < A_LOADS) {
            to_lds16(sized(x_rows, live), to + (uint32_t)(first_x + i * 8 * WN) * kBlock8, x_at + (uint32_t)(i * 8 * WN * row_bytes + kb * kBlock8));
        } else if (i < LOADS) {
            to_lds16(sized(w_rows, live), to + (uint32_t)(BM + first_w + (i - A_LOADS) * 8 * W_WAVES) * kBlock8, w_at + (uint32_t)((i - A_LOADS) * 8 * W_WAVES * row_bytes + kb * kBlock8));
        } else {
            Scales &of = i == LOADS ? scales : more_scales;
            to_lds1(buffer(of.at, live ? of.rows : 0), to + (uint32_t)(NUMBERS + (i - LOADS) * 4 * BM + wave * 256), of.offset);
            of.at += of.step;
        }
    };

    f32x4 acc[TM][TN];
#pragma unroll
    for (int i = 0; i < TM; i++)
#pragma unroll
        for (int j = 0; j < TN; j++) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};

    const int at0 = (quarter ^ (l16 & 7)) * 16, at1 = at0 ^ 64;  // pieces `quarter` and `quarter` + 4 of a row
    const int a_at = (wm * 16 * TM + l16) * kBlock8, b_at = (BM + wn * 16 * TN + l16) * kBlock8;
    auto fragment = [&](const uint8_t *from, int group) {
        const i32x4 low = *reinterpret_cast<const i32x4 *>(from + group * 16 * kBlock8 + at0), high = *reinterpret_cast<const i32x4 *>(from + group * 16 * kBlock8 + at1);
        return (i32x8)__builtin_shufflevector(low, high, 0, 1, 2, 3, 4, 5, 6, 7);
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
            o.sx = scale_words<TM>(s_lds + (wm * 16 + l16) * TM);
        } else if (i <= TN) {
            o.wq[i - 1] = fragment(from + b_at, i - 1);
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
            for (int j = 0; j < TN; j++) wf[j] = exact32<0>(o.wq[j], o.sw.w[j]);
        }
#pragma unroll
        for (int i = 0; i < TM; i++) {
            Exact32 xf;
            if constexpr (EXACT) xf = exact32<FORMAT>(o.xq[i], o.sx.w[i]);
#pragma unroll
            for (int j = 0; j < TN; j++) {
                if constexpr (EXACT) acc[i][j] = mfma16_exact(wf[j], xf, acc[i][j]);
                else acc[i][j] = mfma16<FORMAT>(o.wq[j], o.xq[i], acc[i][j], o.sw.w[j], o.sx.w[i]);
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
                multiply(o, 0, [](int) {});
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
            for (int kb = kb0;; kb += 6) {
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
    T *const y = static_cast<T *>(p.y) + (long)part * p.M * p.N;
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
            if (m >= p.M) continue;
            T *const to = y + (long)m * p.N + n;
            if (n + V <= p.N) {
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

// Few rows: bound by reading QW once.  A workgroup takes some groups of 16 rows of QW and all (at most 16 * MT) rows of X.  Its waves take the blocks of
// K in turn, each lane loads its 2 x 16 bytes of a block of QW itself, AHEAD blocks at a time, and the waves' sums meet in LDS, added up in a
// fixed order.  X lies in LDS as packed numbers (rows 16 bytes more than whole blocks apart, so that 8 rows' pieces meet different banks) and scales:
// INPUT 0 .. 2: fp32 / bf16 / fp16, quantized by the workgroup on the way (a block of a row is 16 lanes of eight); 3: packed.
// One row of 4096 by 4096 x 4096: 5.2-6.0 us with its launch, 16.9 MB at 2.8-3.2 TB/s (through the tiles and a launch of the quantizer 14).  24 rows of
// 2050 (fp16) by 1003: 9.3-10.4 us, bound by every workgroup's conversion of all of X, which costs less than a launch for it alone; 16 waves
// instead of 8 took 5.9-6.4 and 10.9-11.2 us.
struct RowsParams {
    const void *x;
    const uint8_t *sx, *qw, *sw;
    void *y;
    int M, N, K, KB, w_scale_rows, groups_each;
    long ldx;
    Div32 div_kb;
};

// The bound between one launch and quantizer, tiles and join: X in 72 KB of LDS, which up to 16 rows (with 8 KB for the waves' sums) leaves room for two workgroups
// a CU; with 17 to 32 rows the sums take 16 KB, and a CU holds one.  On both sides of it (bf16, by 4096 columns, a pass among others, us):
//   one launch   8 x 4096  8.7   12 x 4096 10.4   17 x 4096 13.0   8 x 8000 15.0   32 x 2176 12.3   32 x 1000 7.4   by 1003 columns 24 x 2050 9.0, 32 x 2050 10.4
//   three        18 x 4096 10.6                                    8 x 9300 12.7   32 x 2304  9.5   33 x 1000 7.0   by 1003 columns 33 x 2050 9.0
// So the largest X in one launch take up to a fifth longer than three launches would; they meet at about 12 rows of 4096.
constexpr int kRowsMost = 32;           // rows of X
constexpr int kRowsLds = 72 << 10;      // bytes of X in LDS
constexpr int kRowsWaves = 8;

__host__ __device__ __forceinline__ int rows_stride(int KB) { return KB * kBlock8 + 16; }
__host__ __device__ __forceinline__ int rows_lds(int M, int KB) { return M * (rows_stride(KB) + KB * 4); }  // numbers, then scales as words [KB][M]

template <int INPUT, int FORMAT, int OUT, int MT>
__global__ __launch_bounds__(64 * kRowsWaves) void linear8_rows(const RowsParams p)
{
    using T = typename Element<OUT>::type;
    constexpr int WAVES = kRowsWaves, AHEAD = 4;
    extern __shared__ __attribute__((aligned(16))) uint8_t packed[];
    __shared__ __attribute__((aligned(16))) float sums[WAVES * MT * 256];
    const int t = threadIdx.x, lane = t % 64, wave = __builtin_amdgcn_readfirstlane(t / 64), l16 = lane % 16, quarter = lane / 16;
    const int stride = rows_stride(p.KB);
    uint32_t *const scales = reinterpret_cast<uint32_t *>(packed + p.M * stride);
    const bool w_rows = p.w_scale_rows == p.N;
    i32x4 w_low[AHEAD], w_high[AHEAD];
    uint32_t w_scale[AHEAD];
    auto load = [&](int n0, int first) {
        const int row = min(n0 + l16, p.N - 1);
        const uint8_t *const w = p.qw + (long)row * p.KB * kBlock8 + quarter * 16, *const sw = p.sw + (w_rows ? row : row / kBlock8);
#pragma unroll
        for (int u = 0; u < AHEAD; u++) {
            const long kb = min(first + u * WAVES, p.KB - 1);
            w_low[u] = *reinterpret_cast<const i32x4 *>(w + kb * kBlock8);
            w_high[u] = *reinterpret_cast<const i32x4 *>(w + kb * kBlock8 + 64);
            w_scale[u] = sw[kb * p.w_scale_rows];
        }
    };
    const int groups = (p.N + 15) / 16, group0 = (int)blockIdx.x * p.groups_each, group1 = min(groups, group0 + p.groups_each);
    load(group0 * 16, wave);

    // X into LDS: blocks in the order of memory, 16 lanes a block, AT_ONCE of them on their way
    constexpr int AT_ONCE = 8, STEP = 64 * WAVES / 16;
    const int blocks = p.M * p.KB;
    for (int first = t / 16; first < blocks; first += AT_ONCE * STEP) {
        using X = typename Element<INPUT == 3 ? 0 : INPUT>::type;
        Words<X> v[AT_ONCE];
#pragma unroll
        for (int u = 0; u < AT_ONCE; u++) {
            const int block = first + u * STEP, m = (int)div32(block, p.div_kb), kb = block - m * p.KB;
            if (block >= blocks) break;
            if constexpr (INPUT == 3) {
                const uint2 w = *reinterpret_cast<const uint2 *>(static_cast<const uint8_t *>(p.x) + (long)block * kBlock8 + l16 * 8);
                v[u].w[0] = w.x, v[u].w[1] = w.y, v[u].w[2] = p.sx[(long)kb * p.M + m];
            } else {
                v[u] = load_words(static_cast<const X *>(p.x) + m * p.ldx, kb * kBlock8 + l16 * 8, p.K);
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
            if (l16 == 0) scales[kb * p.M + m] = byte;
        }
    }
    __syncthreads();

    for (int group = group0; group < group1; group++) {
        const int n0 = group * 16;
        f32x4 acc[MT];
#pragma unroll
        for (int i = 0; i < MT; i++) acc[i] = f32x4{0.f, 0.f, 0.f, 0.f};
        for (int first = wave; first < p.KB; first += AHEAD * WAVES) {
            if (first != wave) load(n0, first);
#pragma unroll
            for (int u = 0; u < AHEAD; u++) {
                const int kb = first + u * WAVES;
                if (kb >= p.KB) break;  // (the same for the whole wave)
                const i32x8 wf = __builtin_shufflevector(w_low[u], w_high[u], 0, 1, 2, 3, 4, 5, 6, 7);
#pragma unroll
                for (int i = 0; i < MT; i++) {
                    const int m = min(i * 16 + l16, p.M - 1);  // (columns past M repeat the last one and are not stored)
                    const uint8_t *const x = packed + m * stride + kb * kBlock8 + quarter * 16;
                    const i32x4 low = *reinterpret_cast<const i32x4 *>(x), high = *reinterpret_cast<const i32x4 *>(x + 64);
                    const i32x8 xf = __builtin_shufflevector(low, high, 0, 1, 2, 3, 4, 5, 6, 7);
                    const uint32_t x_scale = scales[kb * p.M + m];
                    if constexpr (OUT == 0) acc[i] = mfma16_exact(exact32<0>(wf, w_scale[u]), exact32<FORMAT>(xf, x_scale), acc[i]);
                    else acc[i] = mfma16<FORMAT>(wf, xf, acc[i], w_scale[u], x_scale);
                }
            }
        }
        if (group + 1 < group1) load(n0 + 16, wave);  // the next group's first blocks, on their way while the sums meet
#pragma unroll
        for (int i = 0; i < MT; i++) *reinterpret_cast<f32x4 *>(sums + (wave * MT + i) * 256 + l16 * 16 + quarter * 4) = acc[i];
        __syncthreads();
        for (int i = t; i < MT * 256; i += 64 * WAVES) {
            const int m = i / 16, n = n0 + i % 16;
            float sum = sums[i];
#pragma unroll
            for (int k = 1; k < WAVES; k++) sum += sums[k * MT * 256 + i];
            if (m < p.M && n < p.N) static_cast<T *>(p.y)[(long)m * p.N + n] = (T)sum;
        }
        if (group + 1 < group1) __syncthreads();
    }
}

bool rows_fit(int M, int KB) { return M <= kRowsMost && KB <= kRowsLds / kBlock8 && rows_lds(M, KB) <= kRowsLds; }

template <int INPUT, int FORMAT, int OUT> hipError_t launch_rows(RowsParams p, hipStream_t stream)
{
    const int groups = (p.N + 15) / 16;
    p.groups_each = (groups + 511) / 512;  // two workgroups a CU, each with X in its LDS once
    const unsigned workgroups = (unsigned)((groups + p.groups_each - 1) / p.groups_each), lds = (unsigned)rows_lds(p.M, p.KB);
    if (p.M <= 16) linear8_rows<INPUT, FORMAT, OUT, 1><<<workgroups, 64 * kRowsWaves, lds, stream>>>(p);
    else linear8_rows<INPUT, FORMAT, OUT, 2><<<workgroups, 64 * kRowsWaves, lds, stream>>>(p);
    return hipGetLastError();
}

int w_scale_rows(int N, int w_block_rows) { return w_block_rows == 1 ? N : (N + kBlock8 - 1) / kBlock8; }

struct Plan8 {
    int rows, columns;  // of the tile
    int parts, kb_per_part;
    long tiles;
};

// The tile and the parts that K is cut into: the least of what a launch takes by the busiest CU's work.  A step of one of the tiles that a CU holds at
// once takes `alone` us (latency) or, of all its tiles, `among` (throughput), a tile's way out `out`; parts are written in fp32, read and added
// up by a launch of their own.  Constants fitted to every (tile, parts) of 60 products of 33 .. 16384 rows, 64 .. 8192 columns and K on an MI355X;
// what the rule picks takes 0.6 % (16-bit output) and 0.3 % (fp32) longer than the best of them in the mean, at most 14 % (40 x 64 x 8192).
struct TileTimes { int rows, columns, held; double alone, among, out; };

Plan8 plan8(int out, int M, int N, int KB)
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

int threads_of(const Plan8 &plan) { return plan.rows == 256 ? 512 : 256; }

template <int FORMAT, int OUT, bool EXACT> hipError_t launch_tiles(const Plan8 &plan, const TileParams &p, hipStream_t stream)
{
    const unsigned groups = (unsigned)(plan.tiles * plan.parts);
    if constexpr (!EXACT)
        if (plan.rows == 256) {
            linear8_tiles<256, 256, 2, 4, 2, FORMAT, OUT, EXACT><<<groups, threads_of(plan), 0, stream>>>(p);
            return hipGetLastError();
        }
    if (plan.rows == 128) linear8_tiles<128, 128, 2, 2, 2, FORMAT, OUT, EXACT><<<groups, threads_of(plan), 0, stream>>>(p);
    else if (plan.columns == 128) linear8_tiles<64, 128, 2, 2, 3, FORMAT, OUT, EXACT><<<groups, threads_of(plan), 0, stream>>>(p);
    else linear8_tiles<64, 64, 2, 2, 3, FORMAT, OUT, EXACT><<<groups, threads_of(plan), 0, stream>>>(p);
    return hipGetLastError();
}

template <int FORMAT> hipError_t launch_format(int out, const Linear8Args &a, void *workspace, hipStream_t stream)
{
    const int scale_rows = w_scale_rows(a.N, a.w_block_rows);
    if (rows_fit(a.M, a.KB)) {
        const RowsParams p = {a.qx, a.sx, a.qw, a.sw, a.y, a.M, a.N, a.KB * kBlock8, a.KB, scale_rows, 0, 0, make_div32((uint32_t)a.KB)};
        return out == 0 ? launch_rows<3, FORMAT, 0>(p, stream) : out == 1 ? launch_rows<3, FORMAT, 1>(p, stream) : launch_rows<3, FORMAT, 2>(p, stream);
    }
    const Plan8 plan = plan8(out, a.M, a.N, a.KB);
    const int tiles_m = (a.M + plan.rows - 1) / plan.rows, tiles_n = (a.N + plan.columns - 1) / plan.columns;
    TileParams p = {a.qx, a.sx, a.qw, a.sw, plan.parts > 1 ? workspace : a.y, a.M, a.N, a.KB, scale_rows, plan.kb_per_part, tiles_m, tiles_n};
    if (plan.parts == 1)
        return out == 0 ? launch_tiles<FORMAT, 0, true>(plan, p, stream)
                        : out == 1 ? launch_tiles<FORMAT, 1, false>(plan, p, stream) : launch_tiles<FORMAT, 2, false>(plan, p, stream);
    const hipError_t e = out == 0 ? launch_tiles<FORMAT, 0, true>(plan, p, stream) : launch_tiles<FORMAT, 0, false>(plan, p, stream);
    if (e != hipSuccess) return e;
    const long count = (long)a.M * a.N;
    const unsigned joins = (unsigned)((count + 1023) / 1024);
    const float *parts = static_cast<const float *>(workspace);
    if (out == 0) linear8_join<0><<<joins, 256, 0, stream>>>(parts, a.y, count, plan.parts);
    else if (out == 1) linear8_join<1><<<joins, 256, 0, stream>>>(parts, a.y, count, plan.parts);
    else linear8_join<2><<<joins, 256, 0, stream>>>(parts, a.y, count, plan.parts);
    return hipGetLastError();
}

}  // namespace

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
    return x_format == 0 ? launch_format<0>(out_dtype, a, workspace, stream) : launch_format<1>(out_dtype, a, workspace, stream);
}

bool linear8_rows_supported(int M, int K) { return rows_fit(M, blocks8(K)); }

hipError_t launch_linear8_rows(int dtype, const Linear8RowsArgs &a, hipStream_t stream)
{
    const RowsParams p = {a.x, nullptr, a.qw, a.sw, a.y, a.M, a.N, a.K, blocks8(a.K), w_scale_rows(a.N, a.w_block_rows), 0, a.ldx, make_div32((uint32_t)blocks8(a.K))};
    return dtype == 0 ? launch_rows<0, 0, 0>(p, stream) : dtype == 1 ? launch_rows<1, 0, 1>(p, stream) : launch_rows<2, 0, 2>(p, stream);
}

}  // namespace tab
