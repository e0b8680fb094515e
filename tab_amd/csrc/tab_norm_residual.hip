// The norms around a block of a network, with the block's gate and the scaled residual, in one pass over the rows:
//
//   R = alpha X + gate * (Y rms(Y) w_post)      rms(v) = (mean v^2 + eps)^-1/2, a number per row
//   H = R rms(R) w_pre                          the next block's input, plain or as a packed 8-bit operand
//
// and the gradients of X, Y, the gate and both weights.  Everything is fp32 in registers and rounded once where it is stored; H is made
// from R before its rounding.  Memory bound: every row is read once and written once; a row lies in the registers of one group of lanes, in
// runs of eight elements (16 lanes hold a block of 128, so H is packed where it is).  A workgroup takes many rows, so that weights and
// gate are read into registers once.
#include "tab_blocks8.h"
#include "tab_common.h"

namespace tab {

namespace {

template <int GATE, int DTYPE> struct GateElement { using type = typename Element<DTYPE>::type; };
template <int DTYPE> struct GateElement<1, DTYPE> { using type = float; };  // GATE 0: none, 1: fp32, 2: the streams' type

__device__ __forceinline__ float sum_of_wave(float v)
{
#pragma unroll
    for (int d = 1; d < 64; d *= 2) v += __shfl_xor(v, d);
    return v;
}

// Sums over the lanes of a row, in every one of them and in the same order in each.  LANES > 64: one barrier, and `part` may be written again
// only after the next such sum's barrier: two of them take turns (a row's two sums, or every other row's one).
template <int LANES, int N> __device__ __forceinline__ void sum_of_row(float (&v)[N], float *part)
{
#pragma unroll
    for (int i = 0; i < N; i++) v[i] = sum_of_wave(v[i]);
    if constexpr (LANES > 64) {
        const int wave = threadIdx.x / 64;
        if (threadIdx.x % 64 == 0) {
#pragma unroll
            for (int i = 0; i < N; i++) part[wave * N + i] = v[i];
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < N; i++) {
            v[i] = part[i];
#pragma unroll
            for (int w = 1; w < LANES / 64; w++) v[i] += part[w * N + i];
        }
    }
}

struct NormParams {
    const void *x, *y, *gate;
    const float *w_post, *w_pre;
    void *r, *h;
    uint8_t *s;
    int M, D, rows_per_gate, rows_per_group;
    int ldx, ldy;
    float alpha, eps;
};
static_assert(sizeof(NormParams) <= 112, "kernel arguments below 120 bytes");

// Row loop shared by both directions: group g of lanes (a wave, or the workgroup) takes rows [first, end).
template <int LANES> struct RowsOfGroup {
    static constexpr int THREADS = LANES > 256 ? LANES : 256;
    int lane;
    long group;
    __device__ RowsOfGroup() : lane((int)threadIdx.x % LANES), group((long)blockIdx.x * (THREADS / LANES) + threadIdx.x / LANES) {}
};

// OUT: 0 no H, 1 H in the streams' type, 2 H packed (E4M3, 1 x 128 blocks)
template <int DTYPE, int GATE, bool BLOCK, int OUT, int LANES, int RUNS>
__global__ __launch_bounds__((LANES > 256 ? LANES : 256)) void norm_residual(const NormParams p)
{
    using T = typename Element<DTYPE>::type;
    using G = typename GateElement<GATE, DTYPE>::type;
    __shared__ float part[2][32];
    const RowsOfGroup<LANES> rows;
    const long first = rows.group * p.rows_per_group, end = min(first + p.rows_per_group, (long)p.M);
    int at[RUNS], left[RUNS];
    float w_post[RUNS][8], w_pre[RUNS][8], gate[RUNS][8];
#pragma unroll
    for (int c = 0; c < RUNS; c++) {
        at[c] = (c * LANES + rows.lane) * 8;
        left[c] = p.D - at[c];
#pragma unroll
        for (int i = 0; i < 8; i++) w_post[c][i] = w_pre[c][i] = gate[c][i] = 1.f;
        if (BLOCK && p.w_post) load8(p.w_post + at[c], left[c], w_post[c]);
        if (OUT && p.w_pre) load8(p.w_pre + at[c], left[c], w_pre[c]);
    }
    const float over_d = 1.f / (float)p.D;
    long gate_row = -1;
    for (long m = first; m < end; m++) {
        Eight<T> x[RUNS], y[RUNS];
#pragma unroll
        for (int c = 0; c < RUNS; c++) {
            x[c] = load_eight(static_cast<const T *>(p.x) + m * p.ldx + at[c], left[c]);
            if (BLOCK) y[c] = load_eight(static_cast<const T *>(p.y) + m * p.ldy + at[c], left[c]);
        }
        float r[RUNS][8];
        if constexpr (BLOCK) {
            if (GATE) {
                const long wanted = (uint32_t)m / (uint32_t)p.rows_per_gate;
                if (wanted != gate_row) {
                    gate_row = wanted;
#pragma unroll
                    for (int c = 0; c < RUNS; c++) load8(static_cast<const G *>(p.gate) + gate_row * p.D + at[c], left[c], gate[c]);
                }
            }
            float sum[1] = {0.f};
#pragma unroll
            for (int c = 0; c < RUNS; c++)
#pragma unroll
                for (int i = 0; i < 8; i++) sum[0] += (float)y[c].v[i] * (float)y[c].v[i];
            sum_of_row<LANES>(sum, part[OUT ? 0 : m & 1]);
            const float q = rsqrtf(sum[0] * over_d + p.eps);
#pragma unroll
            for (int c = 0; c < RUNS; c++) {
#pragma unroll
                for (int i = 0; i < 8; i++) r[c][i] = p.alpha * (float)x[c].v[i] + gate[c][i] * ((float)y[c].v[i] * q * w_post[c][i]);
                store8(static_cast<T *>(p.r) + m * p.D + at[c], left[c], r[c]);
            }
        } else {
#pragma unroll
            for (int c = 0; c < RUNS; c++)
#pragma unroll
                for (int i = 0; i < 8; i++) r[c][i] = (float)x[c].v[i];
        }
        if constexpr (OUT != 0) {
            float sum[1] = {0.f};
#pragma unroll
            for (int c = 0; c < RUNS; c++)
#pragma unroll
                for (int i = 0; i < 8; i++) sum[0] += i < left[c] ? r[c][i] * r[c][i] : 0.f;
            sum_of_row<LANES>(sum, part[BLOCK ? 1 : m & 1]);
            const float s = rsqrtf(sum[0] * over_d + p.eps);
            const int KB = (p.D + kBlock8 - 1) / kBlock8;
#pragma unroll
            for (int c = 0; c < RUNS; c++) {
                float h[8];
#pragma unroll
                for (int i = 0; i < 8; i++) h[i] = i < left[c] ? r[c][i] * s * w_pre[c][i] : 0.f;
                if constexpr (OUT == 1) {
                    store8(static_cast<T *>(p.h) + m * p.D + at[c], left[c], h);
                } else {
                    uint32_t amax = 0;
#pragma unroll
                    for (int i = 0; i < 8; i++) amax = max(amax, finite_bits(h[i]));
                    const uint32_t byte = scale_byte<0>(max_of_row16(amax));
                    const float inv = inverse_scale(byte);
                    if (at[c] < KB * kBlock8) {
                        const uint2 w = {pack4<0>(h[0], h[1], h[2], h[3], inv), pack4<0>(h[4], h[5], h[6], h[7], inv)};
                        *reinterpret_cast<uint2 *>(static_cast<uint8_t *>(p.h) + m * ((long)KB * kBlock8) + at[c]) = w;
                        if (rows.lane % 16 == 0) p.s[(long)(at[c] / kBlock8) * p.M + m] = (uint8_t)byte;
                    }
                }
            }
        }
    }
}

// ---- gradients -------------------------------------------------------------------------------------------------------
//   a = dH w_pre, p = rms(R):  t = dR + p a - R p^3 mean(R a),  dX = alpha t,  dw_pre = sum over rows of dH R p
//   q = rms(Y), z = Y q w_post:  dgate = sum over the gate's rows of t z,  b = t gate w_post,  dw_post = sum over rows of t gate Y q,
//   dY = q b - Y q^3 mean(Y b)
// p and q are made anew from R and Y, which are here anyway, so the forward pass keeps nothing.  Sums over rows: a group of lanes adds up
// its own rows in registers and leaves them in the workspace, a second launch adds the groups up in a fixed order.

struct NormGradParams {
    const void *dr, *dh, *r, *y, *gate;
    const float *w_post, *w_pre;
    void *dx, *dy, *dgate;
    float *parts;  // [3][groups][D]: dw_post, dw_pre, dgate
    int M, D, rows_per_gate, rows_per_group;
    float alpha, eps;
};
static_assert(sizeof(NormGradParams) <= 112, "kernel arguments below 120 bytes");

// Rows [first, end) of a group.  Gates of few rows: rows_per_group is a multiple of rows_per_gate, a gate's sum ends inside its group.  Gates of
// many rows: a gate is cut into the same number of groups, none of which reaches past it.
__host__ __device__ __forceinline__ bool whole_gates(int rows_per_gate, int rows_per_group) { return rows_per_group % rows_per_gate == 0; }
__host__ __device__ __forceinline__ int groups_per_gate(int rows_per_gate, int rows_per_group) { return (rows_per_gate + rows_per_group - 1) / rows_per_group; }
__host__ __device__ __forceinline__ int groups_of(int M, int rows_per_gate, int rows_per_group)
{
    return whole_gates(rows_per_gate, rows_per_group) ? (int)(((long)M + rows_per_group - 1) / rows_per_group)
                                                      : M / rows_per_gate * groups_per_gate(rows_per_gate, rows_per_group);
}

template <int DTYPE, int GATE, bool BLOCK, int LANES, int RUNS>
__global__ __launch_bounds__((LANES > 256 ? LANES : 256)) void norm_residual_grad(const NormGradParams p)
{
    using T = typename Element<DTYPE>::type;
    using G = typename GateElement<GATE, DTYPE>::type;
    __shared__ float part[2][64];
    const RowsOfGroup<LANES> rows;
    const int groups = groups_of(p.M, p.rows_per_gate, p.rows_per_group);
    if (rows.group >= groups) return;  // (a whole wave of a workgroup without barriers)
    const bool whole = whole_gates(p.rows_per_gate, p.rows_per_group);
    long first = rows.group * p.rows_per_group, end = min(first + p.rows_per_group, (long)p.M);
    if (!whole) {
        const int pieces = groups_per_gate(p.rows_per_gate, p.rows_per_group);
        const long g = rows.group / pieces;
        first = g * p.rows_per_gate + (rows.group - g * pieces) * p.rows_per_group;
        end = min(first + p.rows_per_group, (g + 1) * p.rows_per_gate);
    }
    int at[RUNS], left[RUNS];
    float w_post[RUNS][8], w_pre[RUNS][8], gate[RUNS][8], dw_post[RUNS][8], dw_pre[RUNS][8], dgate[RUNS][8];
#pragma unroll
    for (int c = 0; c < RUNS; c++) {
        at[c] = (c * LANES + rows.lane) * 8;
        left[c] = p.D - at[c];
#pragma unroll
        for (int i = 0; i < 8; i++) {
            w_post[c][i] = w_pre[c][i] = gate[c][i] = 1.f;
            dw_post[c][i] = dw_pre[c][i] = dgate[c][i] = 0.f;
        }
        if (BLOCK && p.w_post) load8(p.w_post + at[c], left[c], w_post[c]);
        if (p.w_pre) load8(p.w_pre + at[c], left[c], w_pre[c]);
    }
    const float over_d = 1.f / (float)p.D;
    long gate_row = -1;
    for (long m = first; m < end; m++) {
        Eight<T> dr[RUNS], dh[RUNS], r[RUNS], y[RUNS];
#pragma unroll
        for (int c = 0; c < RUNS; c++) {
            const long i = m * p.D + at[c];
            dr[c] = load_eight(static_cast<const T *>(p.dr) + i, p.dr ? left[c] : 0);
            dh[c] = load_eight(static_cast<const T *>(p.dh) + i, p.dh ? left[c] : 0);
            r[c] = load_eight(static_cast<const T *>(p.r) + i, p.dh ? left[c] : 0);
            if (BLOCK) y[c] = load_eight(static_cast<const T *>(p.y) + i, left[c]);
        }
        if (BLOCK && GATE) {
            const long wanted = (uint32_t)m / (uint32_t)p.rows_per_gate;
            if (wanted != gate_row) {
                gate_row = wanted;
#pragma unroll
                for (int c = 0; c < RUNS; c++) load8(static_cast<const G *>(p.gate) + gate_row * p.D + at[c], left[c], gate[c]);
            }
        }
        float sum[3] = {0.f, 0.f, 0.f};
#pragma unroll
        for (int c = 0; c < RUNS; c++)
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const float rv = (float)r[c].v[i];
                sum[0] += rv * rv;
                sum[1] += rv * ((float)dh[c].v[i] * w_pre[c][i]);
                if (BLOCK) sum[2] += (float)y[c].v[i] * (float)y[c].v[i];
            }
        sum_of_row<LANES>(sum, part[BLOCK ? 0 : m & 1]);
        const float s = rsqrtf(sum[0] * over_d + p.eps), s3 = s * s * s * (sum[1] * over_d), q = rsqrtf(sum[2] * over_d + p.eps);
        float t[RUNS][8], again[1] = {0.f};
#pragma unroll
        for (int c = 0; c < RUNS; c++) {
            float dx[8];
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const float rv = (float)r[c].v[i], d = (float)dh[c].v[i];
                t[c][i] = (float)dr[c].v[i];
                if (p.dh) {
                    t[c][i] += s * (d * w_pre[c][i]) - rv * s3;
                    dw_pre[c][i] += d * rv * s;
                }
                dx[i] = p.alpha * t[c][i];
                if (BLOCK) {
                    const float yq = (float)y[c].v[i] * q, u = t[c][i] * gate[c][i];
                    dgate[c][i] += t[c][i] * (yq * w_post[c][i]);
                    dw_post[c][i] += u * yq;
                    t[c][i] = u * w_post[c][i];  // b
                    again[0] += (float)y[c].v[i] * t[c][i];
                }
            }
            store8(static_cast<T *>(p.dx) + m * p.D + at[c], left[c], dx);
        }
        if constexpr (BLOCK) {
            sum_of_row<LANES>(again, part[1]);
            const float q3 = q * q * q * (again[0] * over_d);
#pragma unroll
            for (int c = 0; c < RUNS; c++) {
                float dy[8];
#pragma unroll
                for (int i = 0; i < 8; i++) dy[i] = q * t[c][i] - (float)y[c].v[i] * q3;
                store8(static_cast<T *>(p.dy) + m * p.D + at[c], left[c], dy);
            }
            if (GATE && whole && p.dgate && (uint32_t)(m + 1) % (uint32_t)p.rows_per_gate == 0) {
#pragma unroll
                for (int c = 0; c < RUNS; c++) {
                    store8(static_cast<G *>(p.dgate) + gate_row * p.D + at[c], left[c], dgate[c]);
#pragma unroll
                    for (int i = 0; i < 8; i++) dgate[c][i] = 0.f;
                }
            }
        }
    }
    const long slab = (long)groups * p.D, mine = rows.group * p.D;
#pragma unroll
    for (int c = 0; c < RUNS; c++) {
        if (BLOCK) store8(p.parts + mine + at[c], left[c], dw_post[c]);
        store8(p.parts + slab + mine + at[c], left[c], dw_pre[c]);
        if (BLOCK && GATE && !whole) store8(p.parts + 2 * slab + mine + at[c], left[c], dgate[c]);
    }
}

// out[row][d] = sum of the `each` parts of the row: 32 columns by 32 shares of the parts a workgroup, joined in LDS in their order.
struct JoinParams {
    const float *parts;
    void *out;
    int each, D, groups_d;
};
template <int DTYPE> __global__ __launch_bounds__(1024) void norm_grad_join(const JoinParams p)
{
    using T = typename Element<DTYPE>::type;
    __shared__ float sums[32][33];
    const int row = (int)blockIdx.x / p.groups_d, x = threadIdx.x % 32, share = threadIdx.x / 32, d = ((int)blockIdx.x - row * p.groups_d) * 32 + x;
    float sum = 0.f;
    if (d < p.D)
        for (int i = share; i < p.each; i += 32) sum += p.parts[((long)row * p.each + i) * p.D + d];
    sums[share][x] = sum;
    __syncthreads();
    if (share != 0 || d >= p.D) return;
#pragma unroll
    for (int i = 1; i < 32; i++) sum += sums[i][x];
    static_cast<T *>(p.out)[(long)row * p.D + d] = (T)sum;
}

// ---- launches -------------------------------------------------------------------------------------------------------------

constexpr int kLanes[] = {64, 64, 256, 512, 512, 1024}, kRuns[] = {1, 2, 1, 1, 2, 2};  // rows up to 512, 1024, 2048, 4096, 8192, 16384

int shape_of(int D)
{
    int i = 0;
    while (kLanes[i] * kRuns[i] * 8 < D) i++;
    return i;
}

template <int DTYPE, int GATE, bool BLOCK, int OUT> hipError_t launch_shape(NormParams p, hipStream_t stream)
{
    const int shape = shape_of(p.D), per_workgroup = kLanes[shape] == 64 ? 4 : 1;
    // enough groups for the chip, then rows that share the weights' registers
    const long most = 256L * 8 * per_workgroup;
    p.rows_per_group = (int)((p.M + most - 1) / most);
    const long groups = ((long)p.M + p.rows_per_group - 1) / p.rows_per_group;
    const unsigned workgroups = (unsigned)((groups + per_workgroup - 1) / per_workgroup);
    switch (shape) {
    case 0: norm_residual<DTYPE, GATE, BLOCK, OUT, 64, 1><<<workgroups, 256, 0, stream>>>(p); break;
    case 1: norm_residual<DTYPE, GATE, BLOCK, OUT, 64, 2><<<workgroups, 256, 0, stream>>>(p); break;
    case 2: norm_residual<DTYPE, GATE, BLOCK, OUT, 256, 1><<<workgroups, 256, 0, stream>>>(p); break;
    case 3: norm_residual<DTYPE, GATE, BLOCK, OUT, 512, 1><<<workgroups, 512, 0, stream>>>(p); break;
    case 4: norm_residual<DTYPE, GATE, BLOCK, OUT, 512, 2><<<workgroups, 512, 0, stream>>>(p); break;
    default: norm_residual<DTYPE, GATE, BLOCK, OUT, 1024, 2><<<workgroups, 1024, 0, stream>>>(p); break;
    }
    return hipGetLastError();
}

template <int DTYPE, int GATE, bool BLOCK> hipError_t launch_out(const NormParams &p, hipStream_t stream)
{
    if (p.s) return launch_shape<DTYPE, GATE, BLOCK, 2>(p, stream);
    if (p.h) return launch_shape<DTYPE, GATE, BLOCK, 1>(p, stream);
    if constexpr (BLOCK) return launch_shape<DTYPE, GATE, BLOCK, 0>(p, stream);
    return hipErrorInvalidValue;  // (neither R nor H: refused before)
}

template <int DTYPE> hipError_t launch_gate(int gate_dtype, const NormParams &p, hipStream_t stream)
{
    if (!p.y) return launch_out<DTYPE, 0, false>(p, stream);
    if (!p.gate) return launch_out<DTYPE, 0, true>(p, stream);
    if (gate_dtype == 0) return launch_out<DTYPE, 1, true>(p, stream);
    if constexpr (DTYPE != 0) return launch_out<DTYPE, 2, true>(p, stream);
    return hipErrorInvalidValue;  // (a gate of another type: refused before)
}

struct GradPlan {
    int rows_per_group, groups;
};

GradPlan grad_plan(int M, int D, int rows_per_gate)
{
    const long most = 256L * 2 * (kLanes[shape_of(D)] == 64 ? 4 : 1);
    const long rows = (M + most - 1) / most;
    if (rows_per_gate <= rows) {
        const long gates = rows / rows_per_gate;
        const int per = (int)(gates * rows_per_gate);
        return {per, groups_of(M, rows_per_gate, per)};
    }
    const long pieces = (rows_per_gate + rows - 1) / rows;
    const int per = (int)((rows_per_gate + pieces - 1) / pieces);
    return {per, groups_of(M, rows_per_gate, per)};
}

template <int DTYPE, int GATE, bool BLOCK> hipError_t launch_grad_shape(const NormGradParams &p, hipStream_t stream)
{
    const int groups = groups_of(p.M, p.rows_per_gate, p.rows_per_group);
    const int shape = shape_of(p.D), per_workgroup = kLanes[shape] == 64 ? 4 : 1;
    const unsigned workgroups = (unsigned)((groups + per_workgroup - 1) / per_workgroup);
    switch (shape) {
    case 0: norm_residual_grad<DTYPE, GATE, BLOCK, 64, 1><<<workgroups, 256, 0, stream>>>(p); break;
    case 1: norm_residual_grad<DTYPE, GATE, BLOCK, 64, 2><<<workgroups, 256, 0, stream>>>(p); break;
    case 2: norm_residual_grad<DTYPE, GATE, BLOCK, 256, 1><<<workgroups, 256, 0, stream>>>(p); break;
    case 3: norm_residual_grad<DTYPE, GATE, BLOCK, 512, 1><<<workgroups, 512, 0, stream>>>(p); break;
    case 4: norm_residual_grad<DTYPE, GATE, BLOCK, 512, 2><<<workgroups, 512, 0, stream>>>(p); break;
    default: norm_residual_grad<DTYPE, GATE, BLOCK, 1024, 2><<<workgroups, 1024, 0, stream>>>(p); break;
    }
    return hipGetLastError();
}

template <int DTYPE> hipError_t launch_grad_gate(int gate_dtype, const NormGradParams &p, hipStream_t stream)
{
    if (!p.y) return launch_grad_shape<DTYPE, 0, false>(p, stream);
    if (!p.gate) return launch_grad_shape<DTYPE, 0, true>(p, stream);
    if (gate_dtype == 0) return launch_grad_shape<DTYPE, 1, true>(p, stream);
    if constexpr (DTYPE != 0) return launch_grad_shape<DTYPE, 2, true>(p, stream);
    return hipErrorInvalidValue;
}

hipError_t join(int dtype, const float *parts, void *out, int rows, int each, int D, hipStream_t stream)
{
    const JoinParams p = {parts, out, each, D, (D + 31) / 32};
    const unsigned workgroups = (unsigned)rows * (unsigned)p.groups_d;
    if (dtype == 0) norm_grad_join<0><<<workgroups, 1024, 0, stream>>>(p);
    else if (dtype == 1) norm_grad_join<1><<<workgroups, 1024, 0, stream>>>(p);
    else norm_grad_join<2><<<workgroups, 1024, 0, stream>>>(p);
    return hipGetLastError();
}

}  // namespace

hipError_t launch_norm(int dtype, int gate_dtype, const NormArgs &a, hipStream_t stream)
{
    const NormParams p = {a.x, a.y, a.gate, a.w_post, a.w_pre, a.r, a.h, a.s, a.M, a.D, a.rows_per_gate, 0, (int)a.ldx, (int)a.ldy, a.alpha, a.eps};
    return dtype == 0 ? launch_gate<0>(gate_dtype, p, stream) : dtype == 1 ? launch_gate<1>(gate_dtype, p, stream) : launch_gate<2>(gate_dtype, p, stream);
}

size_t norm_grad_workspace(int M, int D, int rows_per_gate) { return 3 * (size_t)grad_plan(M, D, rows_per_gate).groups * (size_t)D * sizeof(float); }

hipError_t launch_norm_grad(int dtype, int gate_dtype, const NormGradArgs &a, float *workspace, hipStream_t stream)
{
    const GradPlan plan = grad_plan(a.M, a.D, a.rows_per_gate);
    const NormGradParams p = {a.dr, a.dh, a.r, a.y, a.gate, a.w_post, a.w_pre, a.dx, a.dy, a.dgate, workspace, a.M, a.D, a.rows_per_gate,
                              plan.rows_per_group, a.alpha, a.eps};
    hipError_t e = dtype == 0 ? launch_grad_gate<0>(gate_dtype, p, stream) : dtype == 1 ? launch_grad_gate<1>(gate_dtype, p, stream) : launch_grad_gate<2>(gate_dtype, p, stream);
    const size_t slab = (size_t)plan.groups * a.D;
    if (e == hipSuccess && a.dw_post) e = join(0, workspace, a.dw_post, 1, plan.groups, a.D, stream);
    if (e == hipSuccess && a.dw_pre) e = join(0, workspace + slab, a.dw_pre, 1, plan.groups, a.D, stream);
    if (e == hipSuccess && a.dgate && !whole_gates(a.rows_per_gate, plan.rows_per_group)) {
        const int gates = a.M / a.rows_per_gate;
        e = join(gate_dtype, workspace + 2 * slab, a.dgate, gates, plan.groups / gates, a.D, stream);
    }
    return e;
}

}  // namespace tab
