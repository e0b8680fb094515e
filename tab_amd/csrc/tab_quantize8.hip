// Quantizers to 8-bit numbers with a power-of-two scale per block of 128 (1 x 128 or 128 x 128), along the rows of X, along
// its columns (X^T packed), or both from one reading of X.
//
//   amax = largest finite |x| of the block;  scale = smallest 2^e >= 2^-126 with amax <= MAX * 2^e;  q = nearest8(x / scale)
//
// Memory bound: reads X once, writes a byte per number and layout.  A large copy reaches 5.1 TB/s on an MI355X (8.4 within the last cache).
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

// Rows of X alone, 1 x 128 blocks: a workgroup takes 32 rows of one block, a row is 16 lanes of eight elements: the largest of a block stays in
// a row of 16 lanes (four exchanges, no LDS), a lane's load is 16 bytes and its store eight.  Small workgroups without a loop, since nothing is kept
// from one block to the next.  bf16 8192 x 8192: 36-38 us, 202 MB at 5.3-5.6 TB/s.
template <int DTYPE, int FORMAT>
__global__ __launch_bounds__(kThreads) void quantize8_rows(const QuantizeParams p)
{
    using T = typename Element<DTYPE>::type;
    const uint32_t tile = blockIdx.x, tile_m = div32(tile, p.div_kb);
    const int kb = (int)(tile - tile_m * (uint32_t)p.KB), tx = threadIdx.x % 16, ty = threadIdx.x / 16, k = kb * kBlock8 + tx * 8;
    Words<T> v[2];
    long row[2];
#pragma unroll
    for (int i = 0; i < 2; i++) {
        row[i] = (long)tile_m * 32 + i * 16 + ty;
        v[i] = load_words(static_cast<const T *>(p.x) + row[i] * p.ldx, k, row[i] < p.M ? p.K : 0);
    }
#pragma unroll
    for (int i = 0; i < 2; i++) {
        uint32_t byte;
        const uint2 w = pack_run<T, FORMAT>(v[i], byte);
        if (row[i] >= p.M) continue;
        *reinterpret_cast<uint2 *>(p.q + row[i] * ((long)p.KB * kBlock8) + k) = w;
        if (tx == 0) p.s[(long)kb * p.M + row[i]] = (uint8_t)byte;
    }
}

// A tile of 128 x 128 that holds infinities or NaN, or rows of less than eight: element by element in fp32, a row
// of the lane's 8 x 8 at a time.
template <int DTYPE, int FORMAT, bool SQUARE>
__device__ __forceinline__ void special_tile(const QuantizeParams &p, uint32_t *transposed, uint32_t *part, uint32_t *bytes)
{
    using T = typename Element<DTYPE>::type;
    const uint32_t tile = blockIdx.x, tile_m = div32(tile, p.div_kb);
    const int kb = (int)(tile - tile_m * (uint32_t)p.KB), t = threadIdx.x, tx = t % 16, ty = t / 16;
    const int k = kb * kBlock8 + tx * 8;
    const long m0 = (long)tile_m * 128, m = m0 + ty * 8;
    const long MB = ((long)p.M + 127) / 128;
    auto row = [&](int i, float (&v)[8]) { load8(static_cast<const T *>(p.x) + (m + i) * p.ldx, k, m + i < p.M ? p.K : 0, v); };
    uint32_t column[8] = {0, 0, 0, 0, 0, 0, 0, 0};
#pragma nounroll
    for (int i = 0; i < 8; i++) {
        float v[8];
        row(i, v);
#pragma unroll
        for (int j = 0; j < 8; j++) column[j] = max(column[j], finite_bits(v[j]));
    }
    uint32_t block_byte = 0;
    if constexpr (SQUARE) {
        uint32_t most = 0;
#pragma unroll
        for (int j = 0; j < 8; j++) most = max(most, column[j]);
        most = max_of_row16(most);
        if (tx == 0) part[ty] = most;
        __syncthreads();
        for (int i = 0; i < 16; i++) most = max(most, part[i]);
        block_byte = scale_byte<FORMAT>(most);
    } else {
#pragma unroll
        for (int j = 0; j < 8; j++) part[ty * 128 + tx * 8 + j] = column[j];
        __syncthreads();
        if (t < 128) {
            uint32_t most = 0;
            for (int i = 0; i < 16; i++) most = max(most, part[i * 128 + t]);
            bytes[t] = scale_byte<FORMAT>(most);
        }
        __syncthreads();
    }
    uint8_t *const flat = reinterpret_cast<uint8_t *>(transposed);
#pragma nounroll
    for (int i = 0; i < 8; i++) {
        float v[8];
        row(i, v);
        uint32_t byte = block_byte, amax = 0;
        if constexpr (!SQUARE) {
#pragma unroll
            for (int j = 0; j < 8; j++) amax = max(amax, finite_bits(v[j]));
            byte = scale_byte<FORMAT>(max_of_row16(amax));
        }
        const float inv = inverse_scale(byte);
        if (p.q && m + i < p.M) {
            *reinterpret_cast<uint2 *>(p.q + (m + i) * ((long)p.KB * kBlock8) + k) =
                uint2{pack4<FORMAT>(v[0], v[1], v[2], v[3], inv), pack4<FORMAT>(v[4], v[5], v[6], v[7], inv)};
            if (!SQUARE && tx == 0) p.s[(long)kb * p.M + m + i] = (uint8_t)byte;
        }
#pragma unroll
        for (int j = 0; j < 8; j++) {
            const int c = tx * 8 + j;
            flat[c * 128 + ty * 8 + i] = (uint8_t)pack4<FORMAT>(v[j], 0.f, 0.f, 0.f, inverse_scale(SQUARE ? block_byte : bytes[c]));
        }
    }
    if (SQUARE && p.q && t == 0) p.s[(long)kb * MB + tile_m] = (uint8_t)block_byte;
    if (!p.qt) return;
    if (SQUARE) {
        if (t == 0) p.st[(long)tile_m * p.KB + kb] = (uint8_t)block_byte;
    } else if (t < 128 && kb * kBlock8 + t < p.K) {
        p.st[(long)tile_m * p.K + kb * kBlock8 + t] = (uint8_t)bytes[t];
    }
    __syncthreads();
    for (int i = t; i < 128 * 8; i += kThreads) {
        const int c = i / 8, g = i % 8;
        if (kb * kBlock8 + c < p.K)
            *reinterpret_cast<uint4 *>(p.qt + (long)(kb * kBlock8 + c) * (MB * kBlock8) + m0 + g * 16) = *reinterpret_cast<const uint4 *>(flat + c * 128 + g * 16);
    }
}

// A tile of 128 x 128: a lane holds 8 rows of 8 columns.  X^T goes through LDS, so that its rows are written as whole cache lines.
// Both layouts leave one reading of X.  What bounded it besides memory was the conversion (an element took its own instructions in each layout):
// two elements an instruction throughout, four waves a SIMD, infinities and NaN in a path of their own that a tile without them skips.
// bf16 8192 x 4096, both layouts: 23 us, 135 MB at 5.8 TB/s (element by element 32); fp32 1531 x 1333 in 128 x 128 blocks 5.4 us (launch and
// one round trip to memory).
template <int DTYPE, int FORMAT, bool SQUARE>
__global__ __launch_bounds__(kThreads) __attribute__((amdgpu_waves_per_eu(4))) void quantize8_tile(const QuantizeParams p)
{
    using T = typename Element<DTYPE>::type;
    constexpr int N = Words<T>::N;
    __shared__ __attribute__((aligned(16))) uint32_t transposed[128 * 32];
    __shared__ __attribute__((aligned(16))) uint32_t part[16 * 128];
    __shared__ uint32_t bytes[128];
    __shared__ uint32_t any_special;
    const uint32_t tile = blockIdx.x, tile_m = div32(tile, p.div_kb);
    const int kb = (int)(tile - tile_m * (uint32_t)p.KB), t = threadIdx.x, tx = t % 16, ty = t / 16;
    const int k = kb * kBlock8 + tx * 8;
    const long m0 = (long)tile_m * 128, m = m0 + ty * 8;
    const long MB = ((long)p.M + 127) / 128;
    if (p.K < 8) return special_tile<DTYPE, FORMAT, SQUARE>(p, transposed, part, bytes);
    // rows past M are the last one's, rows past K its last eight: made zeros below
    Words<T> v[8];
    const int from = min(k, p.K - 8), down = k - from;
#pragma unroll
    for (int i = 0; i < 8; i++) __builtin_memcpy(&v[i], static_cast<const T *>(p.x) + min(m + i, (long)p.M - 1) * p.ldx + from, sizeof(v[i]));
    if (m0 + 128 > p.M || (kb + 1) * kBlock8 > p.K) {
#pragma unroll
        for (int i = 0; i < 8; i++) shift_down(v[i], m + i < p.M ? down : 8);
    }

    // largest of the columns (two a word of 16-bit elements), and whether the tile has to go element by element
    if (t == 0) any_special = 0;
    uint32_t column[N], most = 0;
#pragma unroll
    for (int j = 0; j < N; j++) {
        column[j] = magnitudes<T>(v[0].w[j]);
#pragma unroll
        for (int i = 1; i < 8; i++) column[j] = larger<T>(column[j], magnitudes<T>(v[i].w[j]));
        most = j ? larger<T>(most, column[j]) : column[j];
    }
    if constexpr (sizeof(T) == 2) most = max(most & 0xffffu, most >> 16);
    uint32_t block_byte = 0;
    if constexpr (SQUARE) {
        most = max_of_row16(most);
        if (tx == 0) part[ty] = most;
        __syncthreads();
        most = part[0];
#pragma unroll
        for (int i = 1; i < 16; i++) most = max(most, part[i]);
        if (special<T>(most)) return special_tile<DTYPE, FORMAT, SQUARE>(p, transposed, part + 16, bytes);
        block_byte = scale_byte<FORMAT>(code_bits<T>(most));
    } else {
#pragma unroll
        for (int j = 0; j < N; j++) part[ty * (16 * N) + tx * N + j] = column[j];
        __syncthreads();
        if (special<T>(most)) any_special = 1;
        if (t < 16 * N) {
            uint32_t c = part[t];
#pragma unroll
            for (int i = 1; i < 16; i++) c = larger<T>(c, part[i * (16 * N) + t]);
            if constexpr (sizeof(T) == 4) {
                bytes[t] = scale_byte<FORMAT>(code_bits<T>(c));
            } else {
                bytes[2 * t] = scale_byte<FORMAT>(code_bits<T>(c & 0xffffu));
                bytes[2 * t + 1] = scale_byte<FORMAT>(code_bits<T>(c >> 16));
            }
        }
        __syncthreads();
        if (any_special) return special_tile<DTYPE, FORMAT, SQUARE>(p, transposed, part, bytes);
    }

    if (p.q) {
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const uint32_t byte = SQUARE ? block_byte : scale_byte<FORMAT>(code_bits<T>(max_of_row16(largest(v[i]))));
            if (m + i >= p.M) continue;
            *reinterpret_cast<uint2 *>(p.q + (m + i) * ((long)p.KB * kBlock8) + k) = pack8<T, FORMAT>(v[i], scale_of(byte));
            if (!SQUARE && tx == 0) p.s[(long)kb * p.M + m + i] = (uint8_t)byte;
        }
        if (SQUARE && t == 0) p.s[(long)kb * MB + tile_m] = (uint8_t)block_byte;
    }
    __builtin_amdgcn_sched_barrier(0);

    if (p.qt) {
        if (SQUARE) {
            if (t == 0) p.st[(long)tile_m * p.KB + kb] = (uint8_t)block_byte;
        } else if (t < 128 && kb * kBlock8 + t < p.K) {
            p.st[(long)tile_m * p.K + kb * kBlock8 + t] = (uint8_t)bytes[t];
        }
        // eight bytes (rows m .. m + 7 of one column) at place ty of the column's 16, turned by the column's eighth: the 16
        // columns that a row of lanes writes at once then lie in different banks
#pragma unroll
        for (int j = 0; j < 8; j++) {
            const float scale = scale_of(SQUARE ? block_byte : bytes[tx * 8 + j]);
            Words<T> c;
#pragma unroll
            for (int i = 0; i < N; i++) {
                if constexpr (sizeof(T) == 4) c.w[i] = v[i].w[j];
                else c.w[i] = __builtin_amdgcn_perm(v[2 * i + 1].w[j / 2], v[2 * i].w[j / 2], j % 2 ? 0x07060302u : 0x05040100u);
            }
            *reinterpret_cast<uint2 *>(transposed + (tx * 8 + j) * 32 + (ty ^ tx) * 2) = pack8<T, FORMAT>(c, scale);
            __builtin_amdgcn_sched_barrier(0);  // (all columns at once take registers that are not there)
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
