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

template <int TURN> __device__ __forceinline__ float plus_turned(float v)  // in rows of 16 lanes
{
    return v + __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x120 + TURN, 0xf, 0xf, false));
}
__device__ __forceinline__ float lane_of(float v, int lane) { return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), lane)); }

__device__ __forceinline__ float sum_of_wave(float v)
{
    v = plus_turned<8>(plus_turned<4>(plus_turned<2>(plus_turned<1>(v))));
    return (lane_of(v, 0) + lane_of(v, 16)) + (lane_of(v, 32) + lane_of(v, 48));
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
        // the waves' sums lie in 16 lanes of every wave, and lane 0's total is everybody's
        const int of = threadIdx.x % 16;
#pragma unroll
        for (int i = 0; i < N; i++) {
            const float w = of < LANES / 64 ? part[of * N + i] : 0.f;
            v[i] = lane_of(plus_turned<8>(plus_turned<4>(plus_turned<2>(plus_turned<1>(w)))), 0);
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
    static constexpr int THREADS = LANES > 64 ? LANES : 256;
    int lane;
    long group;
    __device__ RowsOfGroup() : lane((int)threadIdx.x % LANES), group((long)blockIdx.x * (THREADS / LANES) + threadIdx.x / LANES) {}
};

// OUT: 0 no H, 1 H in the streams' type, 2 H packed (E4M3, 1 x 128 blocks)
// bf16 16384 x 4096 with 16 gates: 109-117 us, 537 MB at 4.6-4.9 TB/s (a copy 5.1); one token of 4096 with packed H 2.9 us, its launch.
template <int DTYPE, int GATE, bool BLOCK, int OUT, int LANES, int RUNS>
__global__ __launch_bounds__(RowsOfGroup<LANES>::THREADS) void norm_residual(const NormParams p)
{
    using T = typename Element<DTYPE>::type;
    using G = typename GateElement<GATE, DTYPE>::type;
    constexpr bool AHEAD = RUNS == 1 && sizeof(T) == 2;  // (more takes registers that are not there)
    __shared__ float part[2][32];
    const RowsOfGroup<LANES> rows;
    const long first = rows.group * p.rows_per_group, end = min(first + p.rows_per_group, (long)p.M);
    const bool ragged = p.D != LANES * RUNS * 8;  // rows end before the last lane's last run does
    int at[RUNS], left[RUNS];
    float w_post[RUNS][8], w_pre[RUNS][8], gate[RUNS][8];
#pragma unroll
    for (int c = 0; c < RUNS; c++) {
        at[c] = (c * LANES + rows.lane) * 8;
        left[c] = p.D - at[c];
#pragma unroll
        for (int i = 0; i < 8; i++) w_post[c][i] = w_pre[c][i] = gate[c][i] = 1.f;
        if (BLOCK && p.w_post) load_run8(p.w_post, at[c], p.D, ragged, w_post[c]);
        if (OUT && p.w_pre) load_run8(p.w_pre, at[c], p.D, ragged, w_pre[c]);
    }
    const float over_d = 1.f / (float)p.D;
    long gate_row = -1;
    Words<T> next_x[RUNS], next_y[RUNS];
    auto load = [&](long m) {
#pragma unroll
        for (int c = 0; c < RUNS; c++) {
            next_x[c] = load_run(static_cast<const T *>(p.x) + m * p.ldx, at[c], p.D, ragged);
            if (BLOCK) next_y[c] = load_run(static_cast<const T *>(p.y) + m * p.ldy, at[c], p.D, ragged);
        }
    };
    if (AHEAD && first < end) load(first);
    for (long m = first; m < end; m++) {
        if (!AHEAD) load(m);
        Words<T> x[RUNS], y[RUNS];
#pragma unroll
        for (int c = 0; c < RUNS; c++) {
            x[c] = next_x[c];
            if (BLOCK) y[c] = next_y[c];
        }
        if (AHEAD && m + 1 < end) load(m + 1);  // on its way while this row is worked on
        float r[RUNS][8];
        if constexpr (BLOCK) {
            if (GATE) {
                const long wanted = (uint32_t)m / (uint32_t)p.rows_per_gate;
                if (wanted != gate_row) {
                    gate_row = wanted;
#pragma unroll
                    for (int c = 0; c < RUNS; c++) load_run8(static_cast<const G *>(p.gate) + gate_row * p.D, at[c], p.D, ragged, gate[c]);
                }
            }
            float sum[1] = {0.f};
#pragma unroll
            for (int c = 0; c < RUNS; c++)
#pragma unroll
                for (int i = 0; i < 8; i++) sum[0] += element(y[c], i) * element(y[c], i);
            sum_of_row<LANES>(sum, part[OUT ? 0 : m & 1]);
            const float q = rsqrtf(sum[0] * over_d + p.eps);
#pragma unroll
            for (int c = 0; c < RUNS; c++) {
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    r[c][i] = fmaf(gate[c][i], element(y[c], i) * q * w_post[c][i], p.alpha * element(x[c], i));
                    asm("" : "+v"(r[c][i]));  // in fp32 whatever becomes of it: R has the same bits with and without H
                }
                store8(static_cast<T *>(p.r) + m * p.D + at[c], left[c], r[c]);
            }
        } else {
#pragma unroll
            for (int c = 0; c < RUNS; c++)
#pragma unroll
                for (int i = 0; i < 8; i++) r[c][i] = element(x[c], i);
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
                    Words<float> run;
#pragma unroll
                    for (int i = 0; i < 8; i++) run.w[i] = __float_as_uint(h[i]);
                    uint32_t byte;
                    const uint2 w = pack_run<float, 0>(run, byte);
                    if (at[c] < KB * kBlock8) {
                        *reinterpret_cast<uint2 *>(static_cast<uint8_t *>(p.h) + m * ((long)KB * kBlock8) + at[c]) = w;
                        if (rows.lane % 16 == 0) p.s[(long)(at[c] / kBlock8) * p.M + m] = (uint8_t)byte;
                    }
                }
            }
        }
    }
}

// ---- gradients -------------------------------------------------------------------------------------------------------
//   a = dH w_pre, p = rms(R):  t = dR + p (a - R p^2 mean(R a)),  dX = alpha t,  dw_pre = sum over rows of dH R p
//   q = rms(Y), b = t gate w_post:  dY = q (b - Y q^2 mean(Y b))
// (p^3 and q^3 are outside fp32 for rows beyond 1e13 or, with a small eps, below 1e-13; p p mean(R a), from the right, is as large as a / R)
//   s = sum over a gate's rows of t Y q:  dgate = s w_post,  dw_post = sum over gates of gate s
// p and q are made anew from R and Y, which are here anyway, so the forward pass keeps nothing.  Sums over rows: a group of lanes adds up
// its own rows in registers and leaves them in the workspace, a second launch adds the groups up in a fixed order.
// bf16 16384 x 4096 with 16 gates: 162-167 us, 805 MB at 4.8-5.0 TB/s, and 11-13 for the join; fp32 777 x 1531 with a gate for each row: 14.5 and 4
// (two rows to a group; with three 16.7 and 4).  A group that keeps a gate's, both weights' and their sums' eight columns a lane beside the row's operands needs more
// registers than there are for rows beyond 8192 (two runs a lane: 172 to 591 spilled; bf16 4096 x 16384 480 us, of 157 for its bytes, with a gate a row 910 of 210) and,
// with a gate a row, beyond 2048 in fp32 and 16 bits (16 to 37 spilled; bf16 16384 x 4096 378 us of 210, fp32 470 of 419).  The next row is loaded before this one's sums are taken, as a row alone is all latency.

struct NormGradParams {
    const void *dr, *dh, *r, *y, *gate;
    const float *w_post, *w_pre;
    void *dx, *dy, *dgate;
    float *parts;  // [2][groups][D]: sums for dw_post (WHOLE) or s, and for dw_pre
    int M, D, rows_per_gate, rows_per_group;
    float alpha, eps;
};
static_assert(sizeof(NormGradParams) <= 112, "kernel arguments below 120 bytes");

// Gates of few rows: a group takes whole gates, so that their sums end inside it.  Gates of many rows (and no gate): every gate is cut into the
// same number of groups, none of which reaches past it.
__host__ __device__ __forceinline__ int groups_per_gate(int rows_per_gate, int rows_per_group) { return (int)(((long)rows_per_gate + rows_per_group - 1) / rows_per_group); }
__host__ __device__ __forceinline__ int groups_of(bool whole, int M, int rows_per_gate, int rows_per_group)
{
    return whole ? (int)(((long)M + rows_per_group - 1) / rows_per_group) : M / rows_per_gate * groups_per_gate(rows_per_gate, rows_per_group);
}

template <int DTYPE, int GATE, bool BLOCK, bool WHOLE, int LANES, int RUNS>
__global__ __launch_bounds__(RowsOfGroup<LANES>::THREADS) __attribute__((amdgpu_waves_per_eu(LANES >= 512 ? 4 : 3))) void norm_residual_grad(const NormGradParams p)
{
    using T = typename Element<DTYPE>::type;
    using G = typename GateElement<GATE, DTYPE>::type;
    constexpr bool AHEAD = RUNS == 1 && sizeof(T) == 2;
    __shared__ float part[2][64];
    const RowsOfGroup<LANES> rows;
    const int groups = groups_of(WHOLE, p.M, p.rows_per_gate, p.rows_per_group);
    if (rows.group >= groups) return;  // (a whole wave of a workgroup without barriers)
    long first = rows.group * p.rows_per_group, end = min(first + p.rows_per_group, (long)p.M), gate_row = -1;
    if constexpr (!WHOLE) {
        const int pieces = groups_per_gate(p.rows_per_gate, p.rows_per_group);
        gate_row = rows.group / pieces;
        first = gate_row * p.rows_per_gate + (rows.group - gate_row * pieces) * p.rows_per_group;
        end = min(first + p.rows_per_group, (gate_row + 1) * p.rows_per_gate);
    }
    const bool ragged = p.D != LANES * RUNS * 8;  // rows end before the last lane's last run does
    int at[RUNS], left[RUNS];
    // scale: of t on the way to b, gate w_post (the gate's own while the rows of a WHOLE group change gates: there w_post stays apart)
    float w_pre[RUNS][8], scale[RUNS][8], w_post[WHOLE ? RUNS : 1][8], s[RUNS][8], dw_pre[RUNS][8], dw_post[WHOLE ? RUNS : 1][8];
#pragma unroll
    for (int c = 0; c < RUNS; c++) {
        at[c] = (c * LANES + rows.lane) * 8;
        left[c] = p.D - at[c];
        float post[8];
#pragma unroll
        for (int i = 0; i < 8; i++) {
            w_pre[c][i] = post[i] = scale[c][i] = 1.f;
            s[c][i] = dw_pre[c][i] = 0.f;
        }
        if (p.w_pre) load_run8(p.w_pre, at[c], p.D, ragged, w_pre[c]);
        if constexpr (BLOCK) {
            if (p.w_post) load_run8(p.w_post, at[c], p.D, ragged, post);
            if (GATE && !WHOLE) load_run8(static_cast<const G *>(p.gate) + gate_row * p.D, at[c], p.D, ragged, scale[c]);
        }
#pragma unroll
        for (int i = 0; i < 8; i++) {
            if constexpr (WHOLE) {
                w_post[c][i] = post[i];
                dw_post[c][i] = 0.f;
            } else {
                scale[c][i] *= post[i];
            }
        }
    }
    const float over_d = 1.f / (float)p.D;
    Words<T> next_dr[RUNS], next_dh[RUNS], next_r[RUNS], next_y[RUNS];
    auto load = [&](long m) {
#pragma unroll
        for (int c = 0; c < RUNS; c++) {
            next_dr[c] = next_dh[c] = next_r[c] = Words<T>{};
            if (p.dr) next_dr[c] = load_run(static_cast<const T *>(p.dr) + m * p.D, at[c], p.D, ragged);
            if (p.dh) {
                next_dh[c] = load_run(static_cast<const T *>(p.dh) + m * p.D, at[c], p.D, ragged);
                next_r[c] = load_run(static_cast<const T *>(p.r) + m * p.D, at[c], p.D, ragged);
            }
            if (BLOCK) next_y[c] = load_run(static_cast<const T *>(p.y) + m * p.D, at[c], p.D, ragged);
        }
    };
    if (AHEAD && first < end) load(first);
    for (long m = first; m < end; m++) {
        if (!AHEAD) load(m);
        Words<T> dr[RUNS], dh[RUNS], r[RUNS], y[RUNS];
#pragma unroll
        for (int c = 0; c < RUNS; c++) {
            dr[c] = next_dr[c];
            dh[c] = next_dh[c];
            r[c] = next_r[c];
            if (BLOCK) y[c] = next_y[c];
        }
        if (AHEAD && m + 1 < end) load(m + 1);  // on its way while this row is worked on
        if constexpr (WHOLE) {
            const long wanted = (uint32_t)m / (uint32_t)p.rows_per_gate;
            if (wanted != gate_row) {
                gate_row = wanted;
#pragma unroll
                for (int c = 0; c < RUNS; c++) load_run8(static_cast<const G *>(p.gate) + gate_row * p.D, at[c], p.D, ragged, scale[c]);
            }
        }
        float sum[3] = {0.f, 0.f, 0.f};
#pragma unroll
        for (int c = 0; c < RUNS; c++)
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const float rv = element(r[c], i);
                sum[0] += rv * rv;
                sum[1] += rv * (element(dh[c], i) * w_pre[c][i]);
                if (BLOCK) sum[2] += element(y[c], i) * element(y[c], i);
            }
        sum_of_row<LANES>(sum, part[BLOCK ? 0 : m & 1]);
        const float p1 = rsqrtf(sum[0] * over_d + p.eps), mean_a = p1 * (p1 * (sum[1] * over_d)), q = rsqrtf(sum[2] * over_d + p.eps);
        float t[RUNS][8], again[1] = {0.f};
#pragma unroll
        for (int c = 0; c < RUNS; c++) {
            float dx[8];
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const float rv = element(r[c], i), d = element(dh[c], i);
                t[c][i] = element(dr[c], i);
                if (p.dh) {
                    t[c][i] += p1 * (d * w_pre[c][i] - rv * mean_a);
                    dw_pre[c][i] += d * rv * p1;
                }
                dx[i] = p.alpha * t[c][i];
                if constexpr (BLOCK) {
                    const float yv = element(y[c], i);
                    s[c][i] += t[c][i] * (yv * q);
                    t[c][i] *= scale[c][i];
                    if constexpr (WHOLE) t[c][i] *= w_post[c][i];
                    again[0] += yv * t[c][i];
                }
            }
            store8(static_cast<T *>(p.dx) + m * p.D + at[c], left[c], dx);
        }
        if constexpr (BLOCK) {
            sum_of_row<LANES>(again, part[1]);
            const float mean_b = q * (q * (again[0] * over_d));
#pragma unroll
            for (int c = 0; c < RUNS; c++) {
                float dy[8];
#pragma unroll
                for (int i = 0; i < 8; i++) dy[i] = q * (t[c][i] - element(y[c], i) * mean_b);
                store8(static_cast<T *>(p.dy) + m * p.D + at[c], left[c], dy);
            }
        }
        if constexpr (WHOLE) {
            if ((uint32_t)(m + 1) % (uint32_t)p.rows_per_gate == 0) {
#pragma unroll
                for (int c = 0; c < RUNS; c++) {
                    float dgate[8];
#pragma unroll
                    for (int i = 0; i < 8; i++) {
                        dgate[i] = s[c][i] * w_post[c][i];
                        dw_post[c][i] += s[c][i] * scale[c][i];
                        s[c][i] = 0.f;
                    }
                    if (p.dgate) store8(static_cast<G *>(p.dgate) + gate_row * p.D + at[c], left[c], dgate);
                }
            }
        }
    }
    const long slab = (long)groups * p.D, mine = rows.group * p.D;
#pragma unroll
    for (int c = 0; c < RUNS; c++) {
        if constexpr (WHOLE) store8(p.parts + mine + at[c], left[c], dw_post[c]);
        else if constexpr (BLOCK) store8(p.parts + mine + at[c], left[c], s[c]);
        store8(p.parts + slab + mine + at[c], left[c], dw_pre[c]);
    }
}

// The groups' sums in their order: 32 columns by 32 shares of the groups a workgroup, joined in LDS.  Job 0 is dw_post, 1 dw_pre, 2 + g gate g.
struct JoinParams {
    const float *parts, *w_post;
    const void *gate;  // groups cut out of gates: s of a group counts gate times for dw_post; null: it counts once
    void *dgate;
    float *dw_post, *dw_pre;
    int groups, pieces, D, columns;  // pieces: groups a gate; columns: workgroups a job
};
template <int GATE_DTYPE> __global__ __launch_bounds__(1024) void norm_grad_join(const JoinParams p)
{
    using G = typename Element<GATE_DTYPE>::type;
    __shared__ float sums[32][33];
    const int job = (int)blockIdx.x / p.columns, x = threadIdx.x % 32, share = threadIdx.x / 32, d = ((int)blockIdx.x - job * p.columns) * 32 + x;
    if ((job == 0 && !p.dw_post) || (job == 1 && !p.dw_pre)) return;
    const int first = job < 2 ? 0 : (job - 2) * p.pieces, count = job < 2 ? p.groups : p.pieces;
    const float *const from = p.parts + ((long)(job == 1 ? p.groups : 0) + first) * p.D + d;
    float sum = 0.f;
    if (d < p.D) {
        if (job == 0 && p.gate) {
#pragma unroll 4
            for (int i = share; i < count; i += 32) sum += from[(long)i * p.D] * (float)static_cast<const G *>(p.gate)[(long)(i / p.pieces) * p.D + d];
        } else {
#pragma unroll 4
            for (int i = share; i < count; i += 32) sum += from[(long)i * p.D];
        }
    }
    sums[share][x] = sum;
    __syncthreads();
    if (share != 0 || d >= p.D) return;
#pragma unroll
    for (int i = 1; i < 32; i++) sum += sums[i][x];
    if (job == 0) p.dw_post[d] = sum;
    else if (job == 1) p.dw_pre[d] = sum;
    else static_cast<G *>(p.dgate)[(long)(job - 2) * p.D + d] = (G)(p.w_post ? sum * p.w_post[d] : sum);
}

// ---- launches -------------------------------------------------------------------------------------------------------------

// Lanes of a row by its width, a run of eight elements each up to 8192 (16 waves a CU all the same), two beyond.
constexpr int kWidths[] = {512, 1024, 2048, 4096, 8192, 16384}, kLanes[] = {64, 128, 256, 512, 1024, 1024};

int shape_of(int D)
{
    int i = 0;
    while (kWidths[i] < D) i++;
    return i;
}

// Groups that the chip holds at once
long groups_at_once(int shape) { return 256L * (16 * 64 / kLanes[shape]); }
unsigned workgroups_of(int shape, long groups) { return (unsigned)(kLanes[shape] == 64 ? (groups + 3) / 4 : groups); }

template <int DTYPE, int GATE, bool BLOCK, int OUT> hipError_t launch_shape(NormParams p, hipStream_t stream)
{
    const int shape = shape_of(p.D);
    // no more groups than twice what the chip holds: a group's rows share the weights' registers
    const long most = 2 * groups_at_once(shape);
    p.rows_per_group = (int)((p.M + most - 1) / most);
    const unsigned workgroups = workgroups_of(shape, ((long)p.M + p.rows_per_group - 1) / p.rows_per_group);
    switch (shape) {
    case 0: norm_residual<DTYPE, GATE, BLOCK, OUT, 64, 1><<<workgroups, 256, 0, stream>>>(p); break;
    case 1: norm_residual<DTYPE, GATE, BLOCK, OUT, 128, 1><<<workgroups, 128, 0, stream>>>(p); break;
    case 2: norm_residual<DTYPE, GATE, BLOCK, OUT, 256, 1><<<workgroups, 256, 0, stream>>>(p); break;
    case 3: norm_residual<DTYPE, GATE, BLOCK, OUT, 512, 1><<<workgroups, 512, 0, stream>>>(p); break;
    case 4: norm_residual<DTYPE, GATE, BLOCK, OUT, 1024, 1><<<workgroups, 1024, 0, stream>>>(p); break;
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
    bool whole;
};

GradPlan grad_plan(bool gate, int M, int D, int rows_per_gate)
{
    // as many groups as the chip holds at once, but two rows in each (one where M is odd) before there are more than CUs: every group writes 2 D sums
    const long held = groups_at_once(shape_of(D)), few = M > 512 ? ((long)M + 1) / 2 : 256, most = held < few ? held : few, rows = (M + most - 1) / most;
    const bool whole = gate && rows_per_gate <= rows;
    // (at least one row a group and, for pieces, as even as they come)
    const long pieces = whole ? 1 : (rows_per_gate + rows - 1) / rows;
    const int per = (int)(whole ? rows / rows_per_gate * rows_per_gate : (rows_per_gate + pieces - 1) / pieces);
    return {per, groups_of(whole, M, rows_per_gate, per), whole};
}

template <int DTYPE, int GATE, bool BLOCK, bool WHOLE> hipError_t launch_grad_shape(const NormGradParams &p, int groups, hipStream_t stream)
{
    const int shape = shape_of(p.D);
    const unsigned workgroups = workgroups_of(shape, groups);
    switch (shape) {
    case 0: norm_residual_grad<DTYPE, GATE, BLOCK, WHOLE, 64, 1><<<workgroups, 256, 0, stream>>>(p); break;
    case 1: norm_residual_grad<DTYPE, GATE, BLOCK, WHOLE, 128, 1><<<workgroups, 128, 0, stream>>>(p); break;
    case 2: norm_residual_grad<DTYPE, GATE, BLOCK, WHOLE, 256, 1><<<workgroups, 256, 0, stream>>>(p); break;
    case 3: norm_residual_grad<DTYPE, GATE, BLOCK, WHOLE, 512, 1><<<workgroups, 512, 0, stream>>>(p); break;
    case 4: norm_residual_grad<DTYPE, GATE, BLOCK, WHOLE, 1024, 1><<<workgroups, 1024, 0, stream>>>(p); break;
    default: norm_residual_grad<DTYPE, GATE, BLOCK, WHOLE, 1024, 2><<<workgroups, 1024, 0, stream>>>(p); break;
    }
    return hipGetLastError();
}

template <int DTYPE, int GATE> hipError_t launch_grad_whole(const NormGradParams &p, const GradPlan &plan, hipStream_t stream)
{
    return plan.whole ? launch_grad_shape<DTYPE, GATE, true, true>(p, plan.groups, stream) : launch_grad_shape<DTYPE, GATE, true, false>(p, plan.groups, stream);
}

template <int DTYPE> hipError_t launch_grad_gate(int gate_dtype, const NormGradParams &p, const GradPlan &plan, hipStream_t stream)
{
    if (!p.y) return launch_grad_shape<DTYPE, 0, false, false>(p, plan.groups, stream);
    if (!p.gate) return launch_grad_shape<DTYPE, 0, true, false>(p, plan.groups, stream);
    if (gate_dtype == 0) return launch_grad_whole<DTYPE, 1>(p, plan, stream);
    if constexpr (DTYPE != 0) return launch_grad_whole<DTYPE, 2>(p, plan, stream);
    return hipErrorInvalidValue;  // (a gate of another type: refused before)
}

}  // namespace

hipError_t launch_norm(int dtype, int gate_dtype, const NormArgs &a, hipStream_t stream)
{
    const NormParams p = {a.x, a.y, a.gate, a.w_post, a.w_pre, a.r, a.h, a.s, a.M, a.D, a.rows_per_gate, 0, (int)a.ldx, (int)a.ldy, a.alpha, a.eps};
    return dtype == 0 ? launch_gate<0>(gate_dtype, p, stream) : dtype == 1 ? launch_gate<1>(gate_dtype, p, stream) : launch_gate<2>(gate_dtype, p, stream);
}

size_t norm_grad_workspace(bool gate, int M, int D, int rows_per_gate) { return 2 * (size_t)grad_plan(gate, M, D, rows_per_gate).groups * (size_t)D * sizeof(float); }

hipError_t launch_norm_grad(int dtype, int gate_dtype, const NormGradArgs &a, float *workspace, hipStream_t stream)
{
    const GradPlan plan = grad_plan(a.gate != nullptr, a.M, a.D, a.rows_per_gate);
    const NormGradParams p = {a.dr, a.dh, a.r, a.y, a.gate, a.w_post, a.w_pre, a.dx, a.dy, a.dgate, workspace, a.M, a.D, a.rows_per_gate,
                              plan.rows_per_group, a.alpha, a.eps};
    const hipError_t e = dtype == 0 ? launch_grad_gate<0>(gate_dtype, p, plan, stream) : dtype == 1 ? launch_grad_gate<1>(gate_dtype, p, plan, stream)
                                                                                                    : launch_grad_gate<2>(gate_dtype, p, plan, stream);
    const bool gates = a.dgate && !plan.whole;
    if (e != hipSuccess || (!a.dw_post && !a.dw_pre && !gates)) return e;
    const int columns = (a.D + 31) / 32;
    const JoinParams j = {workspace, a.w_post, plan.whole ? nullptr : a.gate, a.dgate, a.dw_post, a.dw_pre, plan.groups,
                          plan.whole ? 1 : groups_per_gate(a.rows_per_gate, plan.rows_per_group), a.D, columns};
    const unsigned workgroups = (unsigned)columns * (unsigned)(2 + (gates ? a.M / a.rows_per_gate : 0));
    if (gate_dtype == 0) norm_grad_join<0><<<workgroups, 1024, 0, stream>>>(j);
    else if (gate_dtype == 1) norm_grad_join<1><<<workgroups, 1024, 0, stream>>>(j);
    else norm_grad_join<2><<<workgroups, 1024, 0, stream>>>(j);
    return hipGetLastError();
}

}  // namespace tab
