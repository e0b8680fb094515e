// 8-bit numbers with a power-of-two scale per block of 128: formats, element types and the arithmetic that the quantizers,
// the 8-bit product and the norms share.
//
// A packed operand of an R x K matrix is Q, 8-bit numbers [R][128 * ceil(K / 128)] with zeros past K, and S, E8M0 bytes
// [ceil(K / 128)][R] (a block is 128 numbers of one row) or [ceil(K / 128)][ceil(R / 128)] (128 x 128): what it stands for
// is Q[r][k] * 2^(S - 127).
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace tab {

constexpr int kBlock8 = 128;  // numbers under one scale, and a cache line of them

constexpr int blocks8(int K) { return (int)(((long)K + kBlock8 - 1) / kBlock8); }

// Element types, TAB_F32 / TAB_BF16 / TAB_F16 of the C ABI.
template <int DTYPE> struct Element;
template <> struct Element<0> { using type = float; };
template <> struct Element<1> { using type = __bf16; };
template <> struct Element<2> { using type = _Float16; };

// Eight elements as a lane loads and stores them: 16-byte accesses at the elements' own alignment, which the memory pipeline takes at full
// rate inside a cache line, so odd widths and row strides need no code of their own.
template <typename T> struct __attribute__((packed, aligned(sizeof(T)))) Eight { T v[8]; };

// Eight neighbours as they lie in memory: four words of two 16-bit elements, or eight of one.
template <typename T> struct Words { static constexpr int N = 2 * (int)sizeof(T); uint32_t w[N]; };

// Element i becomes element i + n, zeros behind the last; n = 0 .. 7, all zeros from 8 on.
template <typename T> __device__ __forceinline__ void shift_down(Words<T> &v, int n)
{
    constexpr int N = Words<T>::N, PER = 4 / (int)sizeof(T);
#pragma unroll
    for (int step = 4; step >= PER; step /= 2) {
        const bool move = n & step;
#pragma unroll
        for (int i = 0; i < N; i++) v.w[i] = move ? (i + step / PER < N ? v.w[i + step / PER] : 0u) : v.w[i];
    }
    if constexpr (PER == 2) {
        const bool move = n & 1;
#pragma unroll
        for (int i = 0; i < N; i++) v.w[i] = move ? (v.w[i] >> 16 | (i + 1 < N ? v.w[i + 1] << 16 : 0u)) : v.w[i];
    }
#pragma unroll
    for (int i = 0; i < N; i++) v.w[i] = n < 8 ? v.w[i] : 0u;
}

// Elements k .. k + 7 of a row of K, zeros past its end.  The row's last eight are loaded whole and moved into place: element by element the
// ragged end of a row took a dozen loads one after the other.
template <typename T> __device__ __forceinline__ Words<T> load_words(const T *row, int k, int K)
{
    Words<T> v = {};
    const int left = K - k;
    if (left >= 8) {
        __builtin_memcpy(&v, row + k, sizeof(v));
    } else if (left > 0 && K >= 8) {
        __builtin_memcpy(&v, row + (K - 8), sizeof(v));
        shift_down(v, 8 - left);
    } else if (left > 0) {
#pragma unroll
        for (int i = 0; i < 8; i++)
            if (i < left) {
                if constexpr (sizeof(T) == 4) v.w[i] = __float_as_uint(row[k + i]);
                else v.w[i / 2] |= (uint32_t)__builtin_bit_cast(unsigned short, row[k + i]) << 16 * (i % 2);
            }
    }
    return v;
}
// The same for kernels that hold many runs: one load for every lane (the row's last eight where its own reach past the end), and what is
// past the end moved out only where rows end inside a run or before the last lane's (`ragged`).
template <typename T> __device__ __forceinline__ Words<T> load_run(const T *row, int k, int K, bool ragged)
{
    if (K < 8) return load_words(row, k, K);
    Words<T> v;
    const int from = min(k, K - 8);
    __builtin_memcpy(&v, row + from, sizeof(v));
    if (ragged) shift_down(v, k - from);
    return v;
}
template <typename T> __device__ __forceinline__ float element(const Words<T> &v, int i)
{
    if constexpr (sizeof(T) == 4) return __uint_as_float(v.w[i]);
    else return (float)__builtin_bit_cast(T, (unsigned short)(v.w[i / 2] >> 16 * (i % 2)));
}
template <typename T> __device__ __forceinline__ void load8(const T *row, int k, int K, float (&v)[8])
{
    const Words<T> e = load_words(row, k, K);
#pragma unroll
    for (int i = 0; i < 8; i++) v[i] = element(e, i);
}
template <typename T> __device__ __forceinline__ void load_run8(const T *row, int k, int K, bool ragged, float (&v)[8])
{
    const Words<T> e = load_run(row, k, K, ragged);
#pragma unroll
    for (int i = 0; i < 8; i++) v[i] = element(e, i);
}
template <typename T> __device__ __forceinline__ void store8(T *p, int left, const float (&v)[8])
{
    Eight<T> e;
#pragma unroll
    for (int i = 0; i < 8; i++) e.v[i] = (T)v[i];
    if (left >= 8) {
        *reinterpret_cast<Eight<T> *>(p) = e;
    } else {
#pragma unroll
        for (int i = 0; i < 8; i++)
            if (i < left) p[i] = e.v[i];
    }
}

// Magnitude bits of a finite value (their order is the magnitudes'); 0 for infinities and NaN, which set no scale.
__device__ __forceinline__ uint32_t finite_bits(float v)
{
    const uint32_t u = __float_as_uint(v) & 0x7fffffffu;
    return u < 0x7f800000u ? u : 0u;
}

// E8M0 byte of a block whose largest finite magnitude has these bits: the smallest power of two 2^(byte - 127), byte >= 1, with
// magnitude <= MAX * 2^(byte - 127).  MAX is 1.75 * 2^8 (E4M3) or 1.75 * 2^15 (E5M2), so the mantissa decides at 1.75.  A power of two
// makes x / scale exact: a packed number is the nearest 8-bit one to x, with one rounding.  The byte of a block of zeros is 1.
template <int FORMAT> __device__ __forceinline__ uint32_t scale_byte(uint32_t bits)
{
    const int e = (int)(bits >> 23) - (FORMAT == 0 ? 8 : 15) + ((bits & 0x7fffffu) > 0x600000u ? 1 : 0);
    return (uint32_t)(e > 1 ? e : 1);
}

// 2^-(byte - 127), normal for the bytes that scale_byte gives (1 .. 247).
__device__ __forceinline__ float inverse_scale(uint32_t byte) { return __uint_as_float((254u - byte) << 23); }

// Four values times inv as 8-bit numbers, nearest even.  The scale leaves no finite value above the largest number; E4M3 has no
// infinity, there it becomes NaN so that it stays visible.  For blocks that hold infinities or NaN: the others take pack8 below.
template <int FORMAT> __device__ __forceinline__ uint32_t pack4(float a, float b, float c, float d, float inv)
{
    float v[4] = {a * inv, b * inv, c * inv, d * inv};
    if (FORMAT == 0) {
#pragma unroll
        for (int i = 0; i < 4; i++)
            if (__builtin_isinf(v[i])) v[i] = __builtin_nanf("");
        const int low = __builtin_amdgcn_cvt_pk_fp8_f32(v[0], v[1], 0, false);
        return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(v[2], v[3], low, true);
    }
    const int low = __builtin_amdgcn_cvt_pk_bf8_f32(v[0], v[1], 0, false);
    return (uint32_t)__builtin_amdgcn_cvt_pk_bf8_f32(v[2], v[3], low, true);
}

// Blocks of finite elements are packed from the words they lie in, two elements an instruction (masks, packed maxima and conversions that divide
// by the scale): some 3 vector instructions an element in both layouts, where going through fp32 and testing every element for infinities took
// 20 and bound the quantizers (8192 x 4096 bf16 in both layouts: 32.4 us, now 24.6).
typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
typedef short s16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2_ __attribute__((ext_vector_type(2)));
typedef _Float16 f16x2_ __attribute__((ext_vector_type(2)));

// Magnitudes of a word's elements (their codes are in the magnitudes' order) and the larger ones of two words
template <typename T> __device__ __forceinline__ uint32_t magnitudes(uint32_t w) { return w & (sizeof(T) == 4 ? 0x7fffffffu : 0x7fff7fffu); }
template <typename T> __device__ __forceinline__ uint32_t larger(uint32_t a, uint32_t b)
{
    if constexpr (sizeof(T) == 4) return max(a, b);
    else return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(u16x2, a), __builtin_bit_cast(u16x2, b)));
}
template <typename T> __device__ __forceinline__ uint32_t largest(const Words<T> &v)
{
    uint32_t m = magnitudes<T>(v.w[0]);
#pragma unroll
    for (int i = 1; i < Words<T>::N; i++) m = larger<T>(m, magnitudes<T>(v.w[i]));
    return sizeof(T) == 4 ? m : max(m & 0xffffu, m >> 16);
}
// Whether the code of a magnitude is an infinity's or NaN's; the fp32 bits of one that is not
template <typename T> __device__ __forceinline__ bool special(uint32_t code)
{
    return code >= (sizeof(T) == 4 ? 0x7f800000u : __is_same(T, __bf16) ? 0x7f80u : 0x7c00u);
}
template <typename T> __device__ __forceinline__ uint32_t code_bits(uint32_t code)
{
    if constexpr (sizeof(T) == 4) return code;
    else if constexpr (__is_same(T, __bf16)) return code << 16;
    else return __float_as_uint((float)__builtin_bit_cast(_Float16, (unsigned short)code));
}
// 2^(byte - 127)
__device__ __forceinline__ float scale_of(uint32_t byte) { return __uint_as_float(byte << 23); }

// Two words' elements (4 of 16 bits, or the first of two calls' 2 of fp32) over the scale as 8-bit numbers, nearest even
template <typename T, int FORMAT, bool HIGH> __device__ __forceinline__ s16x2 pack2(s16x2 into, uint32_t a, uint32_t b, float scale)
{
    if constexpr (sizeof(T) == 4) {
        if constexpr (FORMAT == 0) return __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(into, __uint_as_float(a), __uint_as_float(b), scale, HIGH);
        else return __builtin_amdgcn_cvt_scalef32_pk_bf8_f32(into, __uint_as_float(a), __uint_as_float(b), scale, HIGH);
    } else if constexpr (__is_same(T, __bf16)) {
        if constexpr (FORMAT == 0) return __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(into, __builtin_bit_cast(bf16x2_, a), scale, HIGH);
        else return __builtin_amdgcn_cvt_scalef32_pk_bf8_bf16(into, __builtin_bit_cast(bf16x2_, a), scale, HIGH);
    } else {
        if constexpr (FORMAT == 0) return __builtin_amdgcn_cvt_scalef32_pk_fp8_f16(into, __builtin_bit_cast(f16x2_, a), scale, HIGH);
        else return __builtin_amdgcn_cvt_scalef32_pk_bf8_f16(into, __builtin_bit_cast(f16x2_, a), scale, HIGH);
    }
}
template <typename T, int FORMAT> __device__ __forceinline__ uint2 pack8(const Words<T> &v, float scale)
{
    s16x2 r[2] = {{0, 0}, {0, 0}};
#pragma unroll
    for (int i = 0; i < 2; i++) {
        constexpr int H = Words<T>::N / 2;  // words of four elements
        r[i] = pack2<T, FORMAT, false>(r[i], v.w[i * H], v.w[i * H + 1], scale);
        if constexpr (H == 4) r[i] = pack2<T, FORMAT, true>(r[i], v.w[i * H + 2], v.w[i * H + 3], scale);
        else r[i] = pack2<T, FORMAT, true>(r[i], v.w[i * H + 1], 0, scale);
    }
    return {__builtin_bit_cast(uint32_t, r[0]), __builtin_bit_cast(uint32_t, r[1])};
}

// Largest of the bits in a row of 16 lanes, in every one of them (row rotations by 1, 2, 4 and 8 lanes).
__device__ __forceinline__ uint32_t max_of_row16(uint32_t v)
{
    v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x121, 0xf, 0xf, false));
    v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x122, 0xf, 0xf, false));
    v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x124, 0xf, 0xf, false));
    return max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x128, 0xf, 0xf, false));
}

// A run of eight of a row's block, 16 lanes a block: the eight numbers and the block's scale byte.
template <typename T, int FORMAT> __device__ __forceinline__ uint2 pack_run(const Words<T> &v, uint32_t &byte)
{
    const uint32_t code = max_of_row16(largest(v));
    if (!special<T>(code)) {
        byte = scale_byte<FORMAT>(code_bits<T>(code));
        return pack8<T, FORMAT>(v, scale_of(byte));
    }
    float f[8];  // (the same for the block's 16 lanes)
    uint32_t amax = 0;
#pragma unroll
    for (int i = 0; i < 8; i++) {
        f[i] = element(v, i);
        amax = max(amax, finite_bits(f[i]));
    }
    byte = scale_byte<FORMAT>(max_of_row16(amax));
    const float inv = inverse_scale(byte);
    return {pack4<FORMAT>(f[0], f[1], f[2], f[3], inv), pack4<FORMAT>(f[4], f[5], f[6], f[7], inv)};
}

// Errors of the C ABI (tab_capi.hip): the message kept for the calling thread, the status returned.
int fail(int status, const char *fmt, ...);
int device_fail(hipError_t e, const char *what);

// ---- launchers (defined in tab_quantize8.hip, tab_linear8.hip and tab_norm_residual.hip) ---------------------------------

struct Quantize8Args {
    const void *x;
    uint8_t *q, *s, *qt, *st;  // either pair may be null
    int M, K;
    long ldx;  // elements between rows of x
    int matrices = 1;  // with blocks of 128 x 128: M x K each, the rows of one behind those of the other
};
// workgroups of a launch (of 256 threads; a launch may hold 2^32 threads)
long quantize8_tiles(int block_rows, bool transposed, int M, int K);
hipError_t launch_quantize8(int dtype, int format, int block_rows, const Quantize8Args &a, hipStream_t stream);

struct Linear8Args {
    const uint8_t *qx, *sx, *qw, *sw;
    void *y;
    int M, N, KB;
    int w_block_rows;  // rows of QW under one scale: 1 or 128
};
constexpr int kBlocks8Most = 65535;   // blocks of K: 256 packed rows stay below 2^31 bytes
constexpr int kRows4Most = 0x1fffffff;  // rows of a weight of 4 bits: their four scale bytes each stay below 2^31 (and what Quantize4 packs in one launch)
size_t linear8_workspace(int out_dtype, int M, int N, int KB);
long linear8_threads(int out_dtype, int M, int N, int KB);  // of the launch
int linear8_way(int out_dtype, int M, int N, int KB);  // 0: few rows; else (the tile's rows + columns) / 2 * 100 + the parts of K
hipError_t launch_linear8(int out_dtype, int x_format, const Linear8Args &a, void *workspace, hipStream_t stream);

// Rows sorted by expert (tab_experts.h): M rows, in QT by blocks of 128 that belong to one expert
hipError_t launch_quantize8_by_expert(int dtype, int format, const Quantize8Args &a, const int *offsets, const int *rows, int E, int x_rows, hipStream_t stream);

// The product that quantizes a few rows of x itself.
bool linear8_rows_supported(int M, int K);
struct Linear8RowsArgs {
    const void *x;
    const uint8_t *qw, *sw;
    void *y;
    int M, N, K;
    int w_block_rows;
    long ldx;
};
hipError_t launch_linear8_rows(int dtype, const Linear8RowsArgs &a, hipStream_t stream);

// Weights of 4 bits (tab_quantize4.hip, tab_linear4.hip): E matrices of M x K, row after row.  A packed one is Q, two E2M1 numbers a byte (the first in the
// low bits), [M][64 * ceil(K / 128)] with zeros past K, and S, E8M0 bytes of groups of 32, [ceil(K / 128)][M][4].
struct Quantize4Args {
    const void *x;
    uint8_t *q, *s;
    int E, M, K;
    long ldx;
};
long quantize4_tiles(long rows, int K);  // workgroups of 256 threads
hipError_t launch_quantize4(int dtype, const Quantize4Args &a, hipStream_t stream);
hipError_t launch_linear4(int out_dtype, const Linear8Args &a, void *workspace, hipStream_t stream);  // (w_block_rows is not read)
bool linear4_rows_supported(int M, int N, int K);
size_t linear4_workspace(int out_dtype, int M, int N, int KB);
hipError_t launch_linear4_rows(int dtype, const Linear8RowsArgs &a, hipStream_t stream);

struct NormArgs {
    const void *x, *y, *gate;      // y and gate may be null
    const float *w_post, *w_pre;   // null: ones
    void *r, *h;                   // null: not wanted; h is the packed operand where s is given
    uint8_t *s;
    int M, D, rows_per_gate;
    long ldx, ldy;
    float alpha, eps;
};
constexpr int kNormWidthMost = 16384;
hipError_t launch_norm(int dtype, int gate_dtype, const NormArgs &a, hipStream_t stream);

struct NormGradArgs {
    const void *dr, *dh;           // either may be null, not both
    const void *r, *y, *gate;      // y and gate may be null
    const float *w_post, *w_pre;
    void *dx, *dy, *dgate;
    float *dw_post, *dw_pre;       // null: not wanted
    int M, D, rows_per_gate;
    float alpha, eps;
};
size_t norm_grad_workspace(bool gate, int M, int D, int rows_per_gate);
hipError_t launch_norm_grad(int dtype, int gate_dtype, const NormGradArgs &a, float *workspace, hipStream_t stream);

}  // namespace tab
