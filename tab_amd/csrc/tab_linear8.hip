// Product of two packed 8-bit operands with power-of-two scales per block of 128,
//   Y[m][n] = sum over kb of 2^(SX[kb][m] + SW[kb][n] - 254) * sum over k in block kb of QX[m][k] QW[n][k].
//
// 16-bit outputs: v_mfma_scale_f32_16x16x128_f8f6f4.  One instruction is a 16 x 16 tile over one block of K, and it takes the E8M0 bytes of its
// 16 rows and 16 columns as operands, so the scales cost no vector instruction and the sums stay in one set of fp32 accumulators.  Inside
// the instruction, products of eight neighbours in K are aligned to the largest of them and keep 13 bits below it (measured): 1.5e-5 of the
// output's size for normal operands, far below the 2^-9 or 2^-12 of the output's own rounding, but not what an fp32 output is for.
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
constexpr uint32_t kNoRow = 0x80000000u;      // an offset past every descriptor here (they end below 2^31): reads zeros

struct TileParams {
    const uint8_t *qx, *sx, *qw, *sw;
    void *y;
    int M, N, KB, w_scale_rows;  // w_scale_rows: scales of QW per block of K, N or ceil(N / 128)
    int kb_per_part;             // blocks of K of a part; with more than one part y is [parts][M][N] fp32
    int tiles_m, tiles_n;
};

template <int FORMAT>
__device__ __forceinline__ f32x4 mfma16(i32x8 w, i32x8 x, f32x4 c, int w_op, int w_scale, int x_op, int x_scale)
{
    // the scales' byte numbers are immediates
#define TAB_MFMA(WO, XO) \
    if (w_op == WO && x_op == XO) return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(w, x, c, 0, FORMAT, WO, w_scale, XO, x_scale)
#define TAB_MFMA4(WO) TAB_MFMA(WO, 0); TAB_MFMA(WO, 1); TAB_MFMA(WO, 2); TAB_MFMA(WO, 3)
    TAB_MFMA4(0);
    TAB_MFMA4(1);
    TAB_MFMA4(2);
    TAB_MFMA4(3);
#undef TAB_MFMA4
#undef TAB_MFMA
    return c;
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

__device__ __forceinline__ void to_lds16(__amdgpu_buffer_rsrc_t rsrc, uint8_t *dst, uint32_t lane_offset, uint32_t offset)
{
    __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, (__attribute__((address_space(3))) void *)dst, 16, lane_offset, offset, 0, 0);
}

template <int N> struct ScaleBytes { uint32_t w[(N + 3) / 4]; };

// N scale bytes of a lane, one for each of its wave's 16-row groups
template <int N> __device__ __forceinline__ ScaleBytes<N> scale_bytes(const uint8_t *p)
{
    ScaleBytes<N> s;
    if constexpr (N == 8) {
        const uint2 v = *reinterpret_cast<const uint2 *>(p);
        s.w[0] = v.x, s.w[1] = v.y;
    } else if constexpr (N == 4) {
        s.w[0] = *reinterpret_cast<const uint32_t *>(p);
    } else {
        static_assert(N == 2, "16-row groups of a wave");
        s.w[0] = *reinterpret_cast<const uint16_t *>(p);
    }
    return s;
}

template <typename T> __device__ __forceinline__ void store4(T *y, f32x4 v, int left)
{
    if (left >= 4) {
        struct __attribute__((packed, aligned(sizeof(T)))) Four { T v[4]; };
        *reinterpret_cast<Four *>(y) = Four{{(T)v[0], (T)v[1], (T)v[2], (T)v[3]}};
    } else {
#pragma unroll
        for (int i = 0; i < 4; i++)
            if (i < left) y[i] = (T)v[i];
    }
}

// A workgroup of WM x WN waves makes a BM x BN tile of Y.  A step is one block of K: 128 bytes of each of the tile's rows, straight
// from global memory into LDS, twice over (the next step's land while this one is multiplied), one barrier a step.  A row is eight
// pieces of 16 bytes; row r has piece g at place g ^ (r & 7), so that the 8 lanes that read at once (8 rows, one piece) meet
// different banks.  Which piece a lane multiplies is free as long as both operands agree, since a block has one scale.
template <int BM, int BN, int WM, int WN, int FORMAT, int OUT, bool EXACT>
__global__ __launch_bounds__(64 * WM * WN) void linear8_tiles(const TileParams p)
{
    using T = typename Element<OUT>::type;
    constexpr int THREADS = 64 * WM * WN, TM = BM / WM / 16, TN = BN / WN / 16, STAGE = (BM + BN) * kBlock8;
    static_assert(BM + BN <= THREADS, "a thread stages one scale");
    constexpr int LOADS = (BM + BN) / 8 / (WM * WN), A_LOADS = BM / 8 / (WM * WN);
    __shared__ __attribute__((aligned(1024))) uint8_t lds[2 * STAGE];
    __shared__ __attribute__((aligned(16))) uint8_t scales[2 * (BM + BN)];

    // the tile: parts of K outermost; every XCD (workgroup number modulo 8) takes one run of the tiles, and a run goes through
    // groups of 8 tiles of rows, so that what its CUs hold at one time reads few rows of either operand
    const uint32_t tiles = (uint32_t)p.tiles_m * (uint32_t)p.tiles_n, part = blockIdx.x / tiles, b = blockIdx.x - part * tiles, share = tiles / 8;
    const uint32_t id = b < share * 8 ? (b & 7) * share + (b >> 3) : b;
    const uint32_t in_group = 8 * (uint32_t)p.tiles_n, group = id / in_group, rest = id - group * in_group;
    const uint32_t rows = min(8u, (uint32_t)p.tiles_m - group * 8), tile_n = rest / rows, tile_m = group * 8 + rest - tile_n * rows;
    const int m0 = (int)tile_m * BM, n0 = (int)tile_n * BN;
    const int kb0 = (int)part * p.kb_per_part, kb1 = min(p.KB, kb0 + p.kb_per_part);

    const int t = threadIdx.x, lane = t % 64, wave = t / 64, wm = wave / WN, wn = wave % WN, l16 = lane % 16, quarter = lane / 16;
    const uint32_t row_bytes = (uint32_t)p.KB * kBlock8;
    const int rows_x = min(BM, p.M - m0), rows_w = min(BN, p.N - n0);
    const __amdgpu_buffer_rsrc_t x_rsrc =
        __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t *>(p.qx) + (long)m0 * row_bytes, 0, (int)(rows_x * row_bytes), kBufferFlags8);
    const __amdgpu_buffer_rsrc_t w_rsrc =
        __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t *>(p.qw) + (long)n0 * row_bytes, 0, (int)(rows_w * row_bytes), kBufferFlags8);
    uint32_t offset[LOADS];
#pragma unroll
    for (int i = 0; i < LOADS; i++) {
        const bool x = i < A_LOADS;
        const int r = ((x ? i : i - A_LOADS) * (WM * WN) + wave) * 8 + lane / 8;
        offset[i] = r < (x ? rows_x : rows_w) ? (uint32_t)r * row_bytes + (uint32_t)((lane % 8) ^ (lane / 8)) * 16 : kNoRow;
    }
    auto load = [&](int buf, int kb) {
#pragma unroll
        for (int i = 0; i < LOADS; i++) {
            const bool x = i < A_LOADS;
            to_lds16(x ? x_rsrc : w_rsrc, lds + buf * STAGE + (x ? 0 : BM * kBlock8) + ((x ? i : i - A_LOADS) * (WM * WN) + wave) * 1024, offset[i],
                     (uint32_t)kb * kBlock8);
        }
    };
    // this thread's scale: of row t of the tile, or of column t - BM; a lane reads those of its 16-row groups side by side
    const bool x_scale = t < BM, stages = t < BM + BN;
    const int r = x_scale ? t : t - BM, group16 = 16 * (x_scale ? TM : TN);
    const int scale_at = (x_scale ? 0 : BM) + r / group16 * group16 + (r % 16) * (x_scale ? TM : TN) + r % group16 / 16;
    const long scale_step = x_scale ? p.M : p.w_scale_rows;
    const uint8_t *scale_from = x_scale ? p.sx + min(m0 + r, p.M - 1) : p.sw + (p.w_scale_rows == p.N ? min(n0 + r, p.N - 1) : min(n0 + r, p.N - 1) / kBlock8);

    f32x4 acc[TM][TN];
#pragma unroll
    for (int i = 0; i < TM; i++)
#pragma unroll
        for (int j = 0; j < TN; j++) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};

    load(0, kb0);
    if (stages) scales[scale_at] = scale_from[kb0 * scale_step];
    for (int kb = kb0; kb < kb1; kb++) {
        const int buf = (kb - kb0) & 1;
        __builtin_amdgcn_s_waitcnt(0);  // this wave's part of the step has landed
        __syncthreads();
        const bool more = kb + 1 < kb1;
        uint8_t next_scale = 0;
        if (more) {
            load(buf ^ 1, kb + 1);
            if (stages) next_scale = scale_from[(kb + 1) * scale_step];
        }
        const uint8_t *a_lds = lds + buf * STAGE + (wm * 16 * TM + l16) * kBlock8, *b_lds = lds + buf * STAGE + (BM + wn * 16 * TN + l16) * kBlock8;
        // pieces `quarter` and `quarter` + 4 of the row
        const int at0 = (quarter ^ (l16 & 7)) * 16, at1 = at0 ^ 64;
        const ScaleBytes<TM> sx = scale_bytes<TM>(scales + buf * (BM + BN) + (wm * 16 + l16) * TM);
        const ScaleBytes<TN> sw = scale_bytes<TN>(scales + buf * (BM + BN) + BM + (wn * 16 + l16) * TN);
        auto fragment = [&](const uint8_t *from, int group) {
            const i32x4 low = *reinterpret_cast<const i32x4 *>(from + group * 16 * kBlock8 + at0), high = *reinterpret_cast<const i32x4 *>(from + group * 16 * kBlock8 + at1);
            return (i32x8)__builtin_shufflevector(low, high, 0, 1, 2, 3, 4, 5, 6, 7);
        };
        if constexpr (EXACT) {
            Exact32 wf[TN];
#pragma unroll
            for (int j = 0; j < TN; j++) wf[j] = exact32<0>(fragment(b_lds, j), sw.w[j / 4] >> 8 * (j % 4) & 255u);
#pragma unroll
            for (int i = 0; i < TM; i++) {
                const Exact32 xf = exact32<FORMAT>(fragment(a_lds, i), sx.w[i / 4] >> 8 * (i % 4) & 255u);
#pragma unroll
                for (int j = 0; j < TN; j++) acc[i][j] = mfma16_exact(wf[j], xf, acc[i][j]);
            }
        } else {
            i32x8 wf[TN];
#pragma unroll
            for (int j = 0; j < TN; j++) wf[j] = fragment(b_lds, j);
#pragma unroll
            for (int i = 0; i < TM; i++) {
                const i32x8 xf = fragment(a_lds, i);
#pragma unroll
                for (int j = 0; j < TN; j++) acc[i][j] = mfma16<FORMAT>(wf[j], xf, acc[i][j], j % 4, (int)sw.w[j / 4], i % 4, (int)sx.w[i / 4]);
            }
        }
        if (more && stages) scales[(buf ^ 1) * (BM + BN) + scale_at] = next_scale;
    }

    // the weights are the instruction's rows: a lane holds four neighbours of one row of Y
    T *y = static_cast<T *>(p.y) + (long)part * p.M * p.N;
#pragma unroll
    for (int i = 0; i < TM; i++) {
        const int m = m0 + (wm * TM + i) * 16 + l16;
        if (m >= p.M) continue;
#pragma unroll
        for (int j = 0; j < TN; j++) {
            const int n = n0 + (wn * TN + j) * 16 + quarter * 4;
            if (n < p.N) store4(y + (long)m * p.N + n, acc[i][j], p.N - n);
        }
    }
}

// The parts of a K that was split over workgroups, added up in their order and rounded once.
template <int OUT> __global__ __launch_bounds__(256) void linear8_join(const float *parts, void *y, long count, int n)
{
    using T = typename Element<OUT>::type;
    const long i = ((long)blockIdx.x * 256 + threadIdx.x) * 4;
    if (i >= count) return;
    if (count % 4 == 0) {
        f32x4 sum = *reinterpret_cast<const f32x4 *>(parts + i);
        for (int k = 1; k < n; k++) sum += *reinterpret_cast<const f32x4 *>(parts + k * count + i);
        store4(static_cast<T *>(y) + i, sum, 4);
    } else {
        for (long j = i; j < min(i + 4, count); j++) {
            float sum = parts[j];
            for (int k = 1; k < n; k++) sum += parts[k * count + j];
            static_cast<T *>(y)[j] = (T)sum;
        }
    }
}

// Few rows: bound by reading QW once, so nothing is shared through LDS on the way.  A workgroup takes 16 rows of QW and all (at most
// 16 * MT) rows of X, its waves take the blocks of K in turn, each lane loads its 2 x 16 bytes of a block itself, and the waves' sums meet
// in LDS, added up in a fixed order.  INPUT 0 .. 2: X is fp32 / bf16 / fp16 and every wave quantizes the blocks it multiplies (a row's block
// lies in 4 lanes); 3: packed.
struct RowsParams {
    const void *x;
    const uint8_t *sx, *qw, *sw;
    void *y;
    int M, N, K, KB, w_scale_rows;
    long ldx;
};

template <typename T> __device__ __forceinline__ void load16(const T *row, int k, int K, bool there, float *v)
{
    float a[8], b[8];
    load8(row + k, there ? K - k : 0, a);
    load8(row + k + 8, there ? K - k - 8 : 0, b);
#pragma unroll
    for (int i = 0; i < 8; i++) v[i] = a[i], v[8 + i] = b[i];
}

template <int INPUT, int FORMAT, int OUT, int MT, int WAVES>
__global__ __launch_bounds__(64 * WAVES) void linear8_rows(const RowsParams p)
{
    using T = typename Element<OUT>::type;
    __shared__ __attribute__((aligned(16))) float sums[WAVES * MT * 256];
    const int t = threadIdx.x, lane = t % 64, wave = t / 64, l16 = lane % 16, quarter = lane / 16;
    const int n0 = blockIdx.x * 16, row_w = min(n0 + l16, p.N - 1);
    const uint8_t *w = p.qw + (long)row_w * p.KB * kBlock8 + quarter * 16;
    const uint8_t *sw = p.sw + (p.w_scale_rows == p.N ? row_w : row_w / kBlock8);
    f32x4 acc[MT];
#pragma unroll
    for (int i = 0; i < MT; i++) acc[i] = f32x4{0.f, 0.f, 0.f, 0.f};
    constexpr int AHEAD = 4;  // blocks of QW that a lane has in flight
    for (int first = wave; first < p.KB; first += AHEAD * WAVES) {
        i32x4 w_low[AHEAD], w_high[AHEAD];
        int w_scale[AHEAD];
#pragma unroll
        for (int u = 0; u < AHEAD; u++) {
            const long kb = min(first + u * WAVES, p.KB - 1);
            w_low[u] = *reinterpret_cast<const i32x4 *>(w + kb * kBlock8);
            w_high[u] = *reinterpret_cast<const i32x4 *>(w + kb * kBlock8 + 64);
            w_scale[u] = sw[kb * p.w_scale_rows];
        }
#pragma unroll
        for (int u = 0; u < AHEAD; u++) {
            const int kb = first + u * WAVES;
            if (kb >= p.KB) break;  // (the same for the whole wave)
            const i32x8 wf = __builtin_shufflevector(w_low[u], w_high[u], 0, 1, 2, 3, 4, 5, 6, 7);
#pragma unroll
            for (int i = 0; i < MT; i++) {
                const int m = i * 16 + l16;
                const bool there = m < p.M;
                i32x8 xf = {0, 0, 0, 0, 0, 0, 0, 0};
                int x_scale = 1;
                if constexpr (INPUT == 3) {
                    if (there) {
                        const uint8_t *x = static_cast<const uint8_t *>(p.x) + ((long)m * p.KB + kb) * kBlock8 + quarter * 16;
                        const i32x4 a = *reinterpret_cast<const i32x4 *>(x), c = *reinterpret_cast<const i32x4 *>(x + 64);
                        xf = __builtin_shufflevector(a, c, 0, 1, 2, 3, 4, 5, 6, 7);
                        x_scale = p.sx[(long)kb * p.M + m];
                    }
                } else {
                    using X = typename Element<INPUT>::type;
                    const X *row = static_cast<const X *>(p.x) + m * p.ldx;
                    float v[32];
                    load16(row, kb * kBlock8 + quarter * 16, p.K, there, v);
                    load16(row, kb * kBlock8 + 64 + quarter * 16, p.K, there, v + 16);
                    uint32_t amax = 0;
#pragma unroll
                    for (int j = 0; j < 32; j++) amax = max(amax, finite_bits(v[j]));
                    amax = max(amax, (uint32_t)__shfl_xor((int)amax, 16));
                    amax = max(amax, (uint32_t)__shfl_xor((int)amax, 32));
                    x_scale = (int)scale_byte<FORMAT>(amax);
                    const float inv = inverse_scale((uint32_t)x_scale);
#pragma unroll
                    for (int j = 0; j < 8; j++) xf[j] = (int)pack4<FORMAT>(v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3], inv);
                }
                if constexpr (OUT == 0) acc[i] = mfma16_exact(exact32<0>(wf, (uint32_t)w_scale[u]), exact32<FORMAT>(xf, (uint32_t)x_scale), acc[i]);
                else acc[i] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(wf, xf, acc[i], 0, FORMAT, 0, w_scale[u], 0, x_scale);
            }
        }
    }
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
}

constexpr int kRowsMost = 32;  // rows of X that linear8_rows takes

template <int INPUT, int FORMAT, int OUT> hipError_t launch_rows(const RowsParams &p, hipStream_t stream)
{
    const unsigned groups = (unsigned)((p.N + 15) / 16);
    if (p.M <= 16) linear8_rows<INPUT, FORMAT, OUT, 1, 8><<<groups, 512, 0, stream>>>(p);
    else linear8_rows<INPUT, FORMAT, OUT, 2, 8><<<groups, 512, 0, stream>>>(p);
    return hipGetLastError();
}

int w_scale_rows(int N, int w_block_rows) { return w_block_rows == 1 ? N : (N + kBlock8 - 1) / kBlock8; }

struct Plan8 {
    int tile, parts, kb_per_part;  // tile: the square tile's edge
};

Plan8 plan8(int out, int M, int N, int KB)
{
    auto tiles = [&](long edge) { return ((M + edge - 1) / edge) * ((N + edge - 1) / edge); };
    const int tile = out != 0 && tiles(256) >= 256 ? 256 : tiles(128) >= 128 ? 128 : 64;
    int parts = 1;
    const long have = tiles(tile);
    while (have * parts * 2 <= 512 && KB / (parts * 2) >= 4) parts *= 2;
    const int per = (KB + parts - 1) / parts;
    return {tile, (KB + per - 1) / per, per};
}

template <int FORMAT, int OUT, bool EXACT> hipError_t launch_tiles(int tile, unsigned groups, const TileParams &p, hipStream_t stream)
{
    if constexpr (!EXACT)
        if (tile == 256) {
            linear8_tiles<256, 256, 2, 4, FORMAT, OUT, EXACT><<<groups, 512, 0, stream>>>(p);
            return hipGetLastError();
        }
    if (tile == 128) linear8_tiles<128, 128, 2, 2, FORMAT, OUT, EXACT><<<groups, 256, 0, stream>>>(p);
    else linear8_tiles<64, 64, 2, 2, FORMAT, OUT, EXACT><<<groups, 256, 0, stream>>>(p);
    return hipGetLastError();
}

template <int FORMAT> hipError_t launch_format(int out, const Linear8Args &a, void *workspace, hipStream_t stream)
{
    const int scale_rows = w_scale_rows(a.N, a.w_block_rows);
    if (a.M <= kRowsMost) {
        const RowsParams p = {a.qx, a.sx, a.qw, a.sw, a.y, a.M, a.N, a.KB * kBlock8, a.KB, scale_rows, 0};
        return out == 0 ? launch_rows<3, FORMAT, 0>(p, stream) : out == 1 ? launch_rows<3, FORMAT, 1>(p, stream) : launch_rows<3, FORMAT, 2>(p, stream);
    }
    const Plan8 plan = plan8(out, a.M, a.N, a.KB);
    const int tiles_m = (a.M + plan.tile - 1) / plan.tile, tiles_n = (a.N + plan.tile - 1) / plan.tile;
    TileParams p = {a.qx, a.sx, a.qw, a.sw, plan.parts > 1 ? workspace : a.y, a.M, a.N, a.KB, scale_rows, plan.kb_per_part, tiles_m, tiles_n};
    const unsigned groups = (unsigned)tiles_m * (unsigned)tiles_n * (unsigned)plan.parts;
    if (plan.parts == 1)
        return out == 0 ? launch_tiles<FORMAT, 0, true>(plan.tile, groups, p, stream)
                        : out == 1 ? launch_tiles<FORMAT, 1, false>(plan.tile, groups, p, stream) : launch_tiles<FORMAT, 2, false>(plan.tile, groups, p, stream);
    const hipError_t e = out == 0 ? launch_tiles<FORMAT, 0, true>(plan.tile, groups, p, stream) : launch_tiles<FORMAT, 0, false>(plan.tile, groups, p, stream);
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
    if (M <= kRowsMost) return 0;
    const Plan8 plan = plan8(out_dtype, M, N, KB);
    return plan.parts > 1 ? (size_t)plan.parts * (size_t)M * (size_t)N * sizeof(float) : 0;
}

long linear8_threads(int out_dtype, int M, int N, int KB)
{
    if (M <= kRowsMost) return ((long)N + 15) / 16 * 512;
    const Plan8 plan = plan8(out_dtype, M, N, KB);
    const long edge = plan.tile;
    return ((M + edge - 1) / edge) * ((N + edge - 1) / edge) * plan.parts * (edge == 256 ? 512 : 256);
}

hipError_t launch_linear8(int out_dtype, int x_format, const Linear8Args &a, void *workspace, hipStream_t stream)
{
    return x_format == 0 ? launch_format<0>(out_dtype, a, workspace, stream) : launch_format<1>(out_dtype, a, workspace, stream);
}

bool linear8_rows_supported(int M) { return M <= kRowsMost; }

hipError_t launch_linear8_rows(int dtype, const Linear8RowsArgs &a, hipStream_t stream)
{
    const RowsParams p = {a.x, nullptr, a.qw, a.sw, a.y, a.M, a.N, a.K, blocks8(a.K), w_scale_rows(a.N, a.w_block_rows), a.ldx};
    return dtype == 0 ? launch_rows<0, 0, 0>(p, stream) : dtype == 1 ? launch_rows<1, 0, 1>(p, stream) : launch_rows<2, 0, 2>(p, stream);
}

}  // namespace tab
