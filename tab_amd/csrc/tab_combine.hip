// The experts' rows back to their tokens: out[t] = sum over j of weights[t][j] Y[places[t][j]], places below zero or past the last row left out, and its
// gradients dY[places[t][j]] = weights[t][j] dout[t] and dweights[t][j] = dout[t] . Y[places[t][j]].  Sums in fp32, in the order of j (and for dweights in one
// order of the lanes), one rounding at the end.  Memory bound: every row is read once.  8192 tokens of 4 rows of 4096, bf16: 67 us, 336 MB at 5.0 TB/s; 777 of 3 rows
// of 1531, fp32: 6.4 us, both gradients 10.7 (latency: a round trip for the places, one for the rows, the sums over the lanes).
#include "tab_blocks8.h"
#include "tab_common.h"
#include "tab_experts.h"

namespace tab {

namespace {

struct CombineParams {
    const void *y;
    const int *places;
    const float *weights;
    void *out;
    int M, k, R, D;
    uint32_t units;  // runs of eight, ceil(D / 8) a token
    Div32 div_unit;
};

// A lane takes a run of eight of a token, four choices on their way at once
template <int Y, int OUT> __global__ __launch_bounds__(256) void combine(const CombineParams p)
{
    using T = typename Element<Y>::type;
    const uint32_t g = blockIdx.x * 256u + threadIdx.x;
    if (g >= p.units) return;
    const int token = (int)div32(g, p.div_unit), d = (int)(g - (uint32_t)token * (uint32_t)((p.D + 7) / 8)) * 8;
    float sum[8] = {};
    for (int first = 0; first < p.k; first += 4) {
        Words<T> v[4];
        float w[4];
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const bool there = first + j < p.k;
            const long at = (long)token * p.k + (there ? first + j : 0);
            const int place = there ? p.places[at] : -1;
            const bool row = place >= 0 && place < p.R;
            w[j] = row ? p.weights ? p.weights[at] : 1.f : 0.f;
            v[j] = load_words(static_cast<const T *>(p.y) + (long)(row ? place : 0) * p.D, d, row ? p.D : 0);
        }
#pragma unroll
        for (int j = 0; j < 4; j++)
#pragma unroll
            for (int i = 0; i < 8; i++) sum[i] = fmaf(w[j], element(v[j], i), sum[i]);
    }
    using O = typename Element<OUT>::type;
    store8(static_cast<O *>(p.out) + (long)token * p.D + d, p.D - d, sum);
}

struct CombineGradParams {
    const void *dout, *y;
    const int *places, *used;
    const float *weights;
    void *dy;
    float *dweights;
    int M, k, R, D;
};

__device__ __forceinline__ float sum_of_wave(float v)
{
#pragma unroll
    for (int step = 32; step; step /= 2) v += __shfl_xor(v, step);
    return v;
}

// WAVES waves take a token; four choices at a time
template <int DTYPE, int WAVES> __global__ __launch_bounds__(256) void combine_grad(const CombineGradParams p)
{
    using T = typename Element<DTYPE>::type;
    __shared__ float sums[4][4];
    const int lane = threadIdx.x % 64, wave = threadIdx.x / 64, part = wave % WAVES;
    const long token = (long)blockIdx.x * (4 / WAVES) + wave / WAVES;
    const bool here = token < p.M;  // (every wave reaches the barriers)
    const T *const dout = static_cast<const T *>(p.dout) + (here ? token : 0) * p.D;
    for (int first = 0; first < p.k; first += 4) {
        long place[4];
        float w[4], dot[4] = {};
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const bool there = here && first + j < p.k;
            const long at = there ? token * p.k + first + j : 0;
            const int row = there ? p.places[at] : -1;
            place[j] = row < p.R ? row : -1;
            w[j] = place[j] >= 0 && p.weights ? p.weights[at] : 1.f;
        }
        for (int d = (part * 64 + lane) * 8; here && d < p.D; d += WAVES * 512) {
            float g[8], v[4][8];
            load8(dout, d, p.D, g);
            if (p.dweights) {
#pragma unroll
                for (int j = 0; j < 4; j++) load8(static_cast<const T *>(p.y) + (place[j] >= 0 ? place[j] : 0) * p.D, d, place[j] >= 0 ? p.D : 0, v[j]);
            }
#pragma unroll
            for (int j = 0; j < 4; j++) {
                if (place[j] < 0) continue;
                if (p.dweights) {
#pragma unroll
                    for (int i = 0; i < 8; i++) dot[j] = fmaf(g[i], v[j][i], dot[j]);
                }
                if (p.dy) {
                    float o[8];
#pragma unroll
                    for (int i = 0; i < 8; i++) o[i] = w[j] * g[i];
                    store8(static_cast<T *>(p.dy) + place[j] * p.D + d, p.D - d, o);
                }
            }
        }
        if (!p.dweights) continue;
#pragma unroll
        for (int j = 0; j < 4; j++) dot[j] = sum_of_wave(dot[j]);
        if constexpr (WAVES > 1) {
            if (lane < 4) sums[wave][lane] = lane == 0 ? dot[0] : lane == 1 ? dot[1] : lane == 2 ? dot[2] : dot[3];
            __syncthreads();
#pragma unroll
            for (int j = 0; j < 4; j++) dot[j] = (sums[0][j] + sums[1][j]) + (sums[2][j] + sums[3][j]);
            __syncthreads();
        }
        if (here && part == 0 && lane < 4 && first + lane < p.k)
            p.dweights[token * p.k + first + lane] = lane == 0 ? dot[0] : lane == 1 ? dot[1] : lane == 2 ? dot[2] : dot[3];
    }
    if (!p.dy || !p.used || !here) return;
    const int used = min(max(*p.used, 0), p.R);  // the rows behind: zeros
    for (long r = token; r < p.R; r += p.M) {
        if (r < used) continue;
        const float zero[8] = {};
        for (int d = (part * 64 + lane) * 8; d < p.D; d += WAVES * 512) store8(static_cast<T *>(p.dy) + r * p.D + d, p.D - d, zero);
    }
}

template <int Y, int OUT> void launch(const CombineParams &p, hipStream_t stream) { combine<Y, OUT><<<(p.units + 255) / 256, 256, 0, stream>>>(p); }

template <int DTYPE> void launch_grad(const CombineGradParams &p, hipStream_t stream)
{
    // a wave a token where there are waves enough or little to do for more
    if (p.M >= 4096 || p.D <= 512) combine_grad<DTYPE, 1><<<(unsigned)(((long)p.M + 3) / 4), 256, 0, stream>>>(p);
    else combine_grad<DTYPE, 4><<<(unsigned)p.M, 256, 0, stream>>>(p);
}

}  // namespace

hipError_t launch_combine(int y, int out, const CombineArgs &a, hipStream_t stream)
{
    const uint32_t each = (uint32_t)((a.D + 7) / 8);
    const CombineParams p = {a.y, a.places, a.weights, a.out, a.M, a.k, a.R, a.D, (uint32_t)a.M * each, make_div32(each)};
    if (y == 0) out == 0 ? launch<0, 0>(p, stream) : out == 1 ? launch<0, 1>(p, stream) : launch<0, 2>(p, stream);
    else y == 1 ? launch<1, 1>(p, stream) : launch<2, 2>(p, stream);
    return hipGetLastError();
}

hipError_t launch_combine_grad(int dtype, const CombineGradArgs &a, hipStream_t stream)
{
    const CombineGradParams p = {a.dout, a.y, a.places, a.used, a.weights, a.dy, a.dweights, a.M, a.k, a.R, a.D};
    dtype == 0 ? launch_grad<0>(p, stream) : dtype == 1 ? launch_grad<1>(p, stream) : launch_grad<2>(p, stream);
    return hipGetLastError();
}

}  // namespace tab
