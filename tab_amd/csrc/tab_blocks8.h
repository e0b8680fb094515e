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

// Eight elements from p, or `left` of them and zeros.
template <typename T> __device__ __forceinline__ Eight<T> load_eight(const T *p, int left)
{
    if (left >= 8) return *reinterpret_cast<const Eight<T> *>(p);
    Eight<T> e;
#pragma unroll
    for (int i = 0; i < 8; i++) e.v[i] = i < left ? p[i] : (T)0.f;
    return e;
}
template <typename T> __device__ __forceinline__ void load8(const T *p, int left, float (&v)[8])
{
    const Eight<T> e = load_eight(p, left);
#pragma unroll
    for (int i = 0; i < 8; i++) v[i] = (float)e.v[i];
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
// infinity, there it becomes NaN so that it stays visible.
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

// Largest of the bits in a row of 16 lanes, in every one of them (row rotations by 1, 2, 4 and 8 lanes).
__device__ __forceinline__ uint32_t max_of_row16(uint32_t v)
{
    v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x121, 0xf, 0xf, false));
    v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x122, 0xf, 0xf, false));
    v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x124, 0xf, 0xf, false));
    return max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x128, 0xf, 0xf, false));
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
size_t linear8_workspace(int out_dtype, int M, int N, int KB);
long linear8_threads(int out_dtype, int M, int N, int KB);  // of the launch
hipError_t launch_linear8(int out_dtype, int x_format, const Linear8Args &a, void *workspace, hipStream_t stream);

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
size_t norm_grad_workspace(int M, int D, int rows_per_gate);
hipError_t launch_norm_grad(int dtype, int gate_dtype, const NormGradArgs &a, float *workspace, hipStream_t stream);

}  // namespace tab
