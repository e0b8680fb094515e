// Quantizer of weights to 4-bit numbers (E2M1: 0, 1/2, 1, 3/2, 2, 3, 4, 6 and their negatives) with a power-of-two scale per group of 32 along the rows.
//
//   amax = largest |w| of the group;  scale = smallest 2^e >= 2^-126 with amax <= 6 * 2^e;  q = nearest4(w / scale), half to even
//
// E2M1 has neither infinities nor NaN: a group that holds one gets the scale byte 255, which stands for NaN, so that it stays visible.
// Memory bound: reads W once, writes 17/32 byte a number.  64 x 2048 x 4096 of bf16 263 us, 1.36 GB at 5.2 TB/s; 8192 x 8192, within the last cache, 25 us.
#include "tab_blocks8.h"
#include "tab_common.h"

namespace tab {

namespace {

constexpr int kThreads = 256;

struct Quantize4Params {
    const void *x;
    uint8_t *q, *s;
    int rows, M, K, KB;  // all rows, and those of one matrix
    long ldx;
    Div32 div_kb, div_m;
};

// E8M0 byte of a group whose largest magnitude has these bits, 6 being 1.5 * 2^2; 1 for a group of zeros
__device__ __forceinline__ uint32_t scale_byte4(uint32_t bits)
{
    const int e = (int)(bits >> 23) - 2 + ((bits & 0x7fffffu) > 0x400000u ? 1 : 0);
    return (uint32_t)(e > 1 ? e : 1);
}

// Eight elements over the scale as eight 4-bit numbers, the first in the low bits
template <typename T> __device__ __forceinline__ uint32_t pack8_of4(const Words<T> &v, float scale)
{
    uint32_t r = 0;
    if constexpr (sizeof(T) == 4) {
        r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, __uint_as_float(v.w[0]), __uint_as_float(v.w[1]), scale, 0);
        r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, __uint_as_float(v.w[2]), __uint_as_float(v.w[3]), scale, 1);
        r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, __uint_as_float(v.w[4]), __uint_as_float(v.w[5]), scale, 2);
        r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, __uint_as_float(v.w[6]), __uint_as_float(v.w[7]), scale, 3);
    } else if constexpr (__is_same(T, __bf16)) {
        r = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(r, __builtin_bit_cast(bf16x2_, v.w[0]), scale, 0);
        r = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(r, __builtin_bit_cast(bf16x2_, v.w[1]), scale, 1);
        r = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(r, __builtin_bit_cast(bf16x2_, v.w[2]), scale, 2);
        r = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(r, __builtin_bit_cast(bf16x2_, v.w[3]), scale, 3);
    } else {
        r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(r, __builtin_bit_cast(f16x2_, v.w[0]), scale, 0);
        r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(r, __builtin_bit_cast(f16x2_, v.w[1]), scale, 1);
        r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(r, __builtin_bit_cast(f16x2_, v.w[2]), scale, 2);
        r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(r, __builtin_bit_cast(f16x2_, v.w[3]), scale, 3);
    }
    return r;
}

// A workgroup takes 32 rows of one block of 128: a row's block is 16 lanes of eight elements, a group four neighbouring lanes.
template <int DTYPE> __global__ __launch_bounds__(kThreads) void quantize4_rows(const Quantize4Params p)
{
    using T = typename Element<DTYPE>::type;
    const uint32_t tile = blockIdx.x, tile_m = div32(tile, p.div_kb);
    const int kb = (int)(tile - tile_m * (uint32_t)p.KB), tx = threadIdx.x % 16, ty = threadIdx.x / 16, k = kb * kBlock8 + tx * 8;
    Words<T> v[2];
    long row[2];
#pragma unroll
    for (int i = 0; i < 2; i++) {
        row[i] = (long)tile_m * 32 + i * 16 + ty;
        v[i] = load_words(static_cast<const T *>(p.x) + row[i] * p.ldx, k, row[i] < p.rows ? p.K : 0);
    }
#pragma unroll
    for (int i = 0; i < 2; i++) {
        uint32_t code = largest(v[i]);
        code = max(code, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)code, 0xb1, 0xf, 0xf, false));  // lanes 1 0 3 2
        code = max(code, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)code, 0x4e, 0xf, 0xf, false));  // lanes 2 3 0 1
        const bool bad = special<T>(code);
        const uint32_t byte = bad ? 255u : scale_byte4(code_bits<T>(code)), numbers = pack8_of4(v[i], bad ? 1.f : scale_of(byte));
        if (row[i] >= p.rows) continue;
        *reinterpret_cast<uint32_t *>(p.q + row[i] * ((long)p.KB * 64) + k / 2) = bad ? 0u : numbers;
        const long e = div32((uint32_t)row[i], p.div_m), m = row[i] - e * p.M;
        if (tx % 4 == 0) p.s[((e * p.KB + kb) * p.M + m) * 4 + tx / 4] = (uint8_t)byte;
    }
}

}  // namespace

long quantize4_tiles(long rows, int K) { return (rows + 31) / 32 * blocks8(K); }

hipError_t launch_quantize4(int dtype, const Quantize4Args &a, hipStream_t stream)
{
    const int KB = blocks8(a.K), rows = a.E * a.M;
    const Quantize4Params p = {a.x, a.q, a.s, rows, a.M, a.K, KB, a.ldx, make_div32((uint32_t)KB), make_div32((uint32_t)a.M)};
    const unsigned tiles = (unsigned)quantize4_tiles(rows, a.K);
    if (dtype == 0) quantize4_rows<0><<<tiles, kThreads, 0, stream>>>(p);
    else if (dtype == 1) quantize4_rows<1><<<tiles, kThreads, 0, stream>>>(p);
    else quantize4_rows<2><<<tiles, kThreads, 0, stream>>>(p);
    return hipGetLastError();
}

}  // namespace tab
