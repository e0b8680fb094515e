// Quantizers to 8-bit numbers with a power-of-two scale per block of 128 (1 x 128 or 128 x 128), along the rows of X, along
// its columns (X^T packed), or both from one reading of X.
//
//   amax = largest finite |x| of the block;  scale = smallest 2^e >= 2^-126 with amax <= MAX * 2^e;  q = nearest8(x / scale)
//
// Memory bound: reads X once, writes a byte per number and layout.
#include "tab_blocks8.h"
#include "tab_common.h"

namespace tab {

namespace {

constexpr int kThreads = 256;

struct QuantizeParams {
    const void *x;
    uint8_t *q, *s, *qt, *st;
    int M, K, KB, tiles;
    long ldx;
    Div32 div_kb;
};

// Rows of X alone, 1 x 128 blocks: a workgroup takes 32 rows of one block, a row is 16 lanes of eight elements.
template <int DTYPE, int FORMAT>
__global__ __launch_bounds__(kThreads) void quantize8_rows(const QuantizeParams p)
{
    using T = typename Element<DTYPE>::type;
    const uint32_t tile = blockIdx.x, tile_m = div32(tile, p.div_kb);
    const int kb = (int)(tile - tile_m * (uint32_t)p.KB), tx = threadIdx.x % 16, ty = threadIdx.x / 16;
    const int k = kb * kBlock8 + tx * 8, left = p.K - k;
    float v[2][8];
    long row[2];
#pragma unroll
    for (int i = 0; i < 2; i++) {
        row[i] = (long)tile_m * 32 + i * 16 + ty;
        load8(static_cast<const T *>(p.x) + row[i] * p.ldx + k, row[i] < p.M ? left : 0, v[i]);
    }
#pragma unroll
    for (int i = 0; i < 2; i++) {
        uint32_t amax = 0;
#pragma unroll
        for (int j = 0; j < 8; j++) amax = max(amax, finite_bits(v[i][j]));
        const uint32_t byte = scale_byte<FORMAT>(max_of_row16(amax));
        const float inv = inverse_scale(byte);
        if (row[i] >= p.M) continue;
        const uint2 w = {pack4<FORMAT>(v[i][0], v[i][1], v[i][2], v[i][3], inv), pack4<FORMAT>(v[i][4], v[i][5], v[i][6], v[i][7], inv)};
        *reinterpret_cast<uint2 *>(p.q + row[i] * ((long)p.KB * kBlock8) + k) = w;
        if (tx == 0) p.s[(long)kb * p.M + row[i]] = (uint8_t)byte;
    }
}

// A tile of 128 x 128: a lane holds 8 rows of 8 columns.  X^T goes through LDS, so that its rows are written as whole cache lines.
template <int DTYPE, int FORMAT, bool SQUARE>
__global__ __launch_bounds__(kThreads) void quantize8_tile(const QuantizeParams p)
{
    using T = typename Element<DTYPE>::type;
    __shared__ __attribute__((aligned(16))) uint32_t transposed[128 * 32];
    __shared__ uint32_t part[16 * 128];
    __shared__ uint32_t bytes[128];
    const uint32_t tile = blockIdx.x, tile_m = div32(tile, p.div_kb);
    const int kb = (int)(tile - tile_m * (uint32_t)p.KB), t = threadIdx.x, tx = t % 16, ty = t / 16;
    const int k = kb * kBlock8 + tx * 8, left = p.K - k;
    const long m0 = (long)tile_m * 128, m = m0 + ty * 8;
    const long MB = ((long)p.M + 127) / 128;
    float v[8][8];
#pragma unroll
    for (int i = 0; i < 8; i++)
        load8(static_cast<const T *>(p.x) + (m + i) * p.ldx + k, m + i < p.M ? left : 0, v[i]);

    uint32_t block_byte = 0;
    if constexpr (SQUARE) {
        uint32_t amax = 0;
#pragma unroll
        for (int i = 0; i < 8; i++)
#pragma unroll
            for (int j = 0; j < 8; j++) amax = max(amax, finite_bits(v[i][j]));
        amax = max_of_row16(amax);
        if (tx == 0) part[ty] = amax;
        __syncthreads();
        amax = 0;
#pragma unroll
        for (int i = 0; i < 16; i++) amax = max(amax, part[i]);
        block_byte = scale_byte<FORMAT>(amax);
    }

    if (p.q) {
#pragma unroll
        for (int i = 0; i < 8; i++) {
            uint32_t byte = block_byte;
            if constexpr (!SQUARE) {
                uint32_t amax = 0;
#pragma unroll
                for (int j = 0; j < 8; j++) amax = max(amax, finite_bits(v[i][j]));
                byte = scale_byte<FORMAT>(max_of_row16(amax));
            }
            if (m + i >= p.M) continue;
            const float inv = inverse_scale(byte);
            const uint2 w = {pack4<FORMAT>(v[i][0], v[i][1], v[i][2], v[i][3], inv), pack4<FORMAT>(v[i][4], v[i][5], v[i][6], v[i][7], inv)};
            *reinterpret_cast<uint2 *>(p.q + (m + i) * ((long)p.KB * kBlock8) + k) = w;
            if (!SQUARE && tx == 0) p.s[(long)kb * p.M + m + i] = (uint8_t)byte;
        }
        if (SQUARE && t == 0) p.s[(long)kb * MB + tile_m] = (uint8_t)block_byte;
    }

    if (p.qt) {
        if constexpr (!SQUARE) {
#pragma unroll
            for (int j = 0; j < 8; j++) {
                uint32_t amax = 0;
#pragma unroll
                for (int i = 0; i < 8; i++) amax = max(amax, finite_bits(v[i][j]));
                part[ty * 128 + tx * 8 + j] = amax;
            }
            __syncthreads();
            if (t < 128) {
                uint32_t amax = 0;
#pragma unroll
                for (int i = 0; i < 16; i++) amax = max(amax, part[i * 128 + t]);
                bytes[t] = scale_byte<FORMAT>(amax);
                if (kb * kBlock8 + t < p.K) p.st[(long)tile_m * p.K + kb * kBlock8 + t] = (uint8_t)bytes[t];
            }
            __syncthreads();
        } else if (t == 0) {
            p.st[(long)tile_m * p.KB + kb] = (uint8_t)block_byte;
        }
        // eight bytes (rows m .. m + 7 of one column) at place ty of the column's 16, turned by the column's eighth: the 16
        // columns that a row of lanes writes at once then lie in different banks
#pragma unroll
        for (int j = 0; j < 8; j++) {
            const float inv = inverse_scale(SQUARE ? block_byte : bytes[tx * 8 + j]);
            const uint2 w = {pack4<FORMAT>(v[0][j], v[1][j], v[2][j], v[3][j], inv), pack4<FORMAT>(v[4][j], v[5][j], v[6][j], v[7][j], inv)};
            *reinterpret_cast<uint2 *>(transposed + (tx * 8 + j) * 32 + (ty ^ tx) * 2) = w;
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const int c = i * 32 + t / 8, turn = c / 8, g = t % 8;
            uint4 w = *reinterpret_cast<const uint4 *>(transposed + c * 32 + (g ^ (turn >> 1)) * 4);
            if (turn & 1) w = {w.z, w.w, w.x, w.y};
            if (kb * kBlock8 + c < p.K) *reinterpret_cast<uint4 *>(p.qt + (long)(kb * kBlock8 + c) * (MB * kBlock8) + m0 + g * 16) = w;
        }
    }
}

template <int DTYPE, int FORMAT>
hipError_t launch(int block_rows, const QuantizeParams &p, hipStream_t stream)
{
    if (block_rows == 1 && !p.qt) quantize8_rows<DTYPE, FORMAT><<<p.tiles, kThreads, 0, stream>>>(p);
    else if (block_rows == 1) quantize8_tile<DTYPE, FORMAT, false><<<p.tiles, kThreads, 0, stream>>>(p);
    else quantize8_tile<DTYPE, FORMAT, true><<<p.tiles, kThreads, 0, stream>>>(p);
    return hipGetLastError();
}

template <int DTYPE> hipError_t launch(int format, int block_rows, const QuantizeParams &p, hipStream_t stream)
{
    return format == 0 ? launch<DTYPE, 0>(block_rows, p, stream) : launch<DTYPE, 1>(block_rows, p, stream);
}

}  // namespace

long quantize8_tiles(int block_rows, bool transposed, int M, int K)
{
    const long rows = block_rows == 1 && !transposed ? 32 : 128;
    return ((long)M + rows - 1) / rows * blocks8(K);
}

hipError_t launch_quantize8(int dtype, int format, int block_rows, const Quantize8Args &a, hipStream_t stream)
{
    const int KB = blocks8(a.K);
    const QuantizeParams p = {a.x, a.q, a.s, a.qt, a.st, a.M, a.K, KB, (int)quantize8_tiles(block_rows, a.qt != nullptr, a.M, a.K), a.ldx,
                              make_div32((uint32_t)KB)};
    return dtype == 0 ? launch<0>(format, block_rows, p, stream) : dtype == 1 ? launch<1>(format, block_rows, p, stream) : launch<2>(format, block_rows, p, stream);
}

}  // namespace tab
