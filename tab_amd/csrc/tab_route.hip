// The router of a layer of experts: the k experts with the largest logits of each token, their weights, and the order of the rows by expert.
//
//   weights = softmax of the logits, over the k chosen ones (normalize) or over all, of the chosen ones;  rows sorted by (expert, token), so that the
//   same logits give the same order.  Gradient, with g of the weights w: dlogit_e = p_e (g_e - sum over j of g_j w_j), p the softmax that the
//   weights are of, g_e zero where e was not chosen.
//
// An expert at -inf is closed and never chosen; a token with fewer than k open experts has -1 and the weight 0 in the remaining places.  NaN counts as the largest
// logit, so that it stays visible: the weights of its token become NaN.  Ties go to the lower index; -0 and 0 are equal.
//
// Bound by latency: a choice is one maximum over the wave after the other, and a row's place one exchange through LDS after the other.  16 tokens, 64 experts, 4
// choices: one launch of 4.0 us; 16384 tokens (bf16) 8.0 + 8.2, their gradient 5.4 (2 MB read, 0.9 MB of whole numbers written).
#include "tab_blocks8.h"
#include "tab_common.h"
#include "tab_experts.h"

namespace tab {

namespace {

constexpr int kThreads = 1024, kWaves = kThreads / 64;

// A code in the order of the logits; 0 for -inf and for what is past the last expert
__device__ __forceinline__ uint32_t order_code(float v)
{
    const uint32_t u = __float_as_uint(v + 0.f);  // (-0 becomes 0)
    if (v != v) return 0xffffffffu;
    return u == 0xff800000u ? 0u : u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float value_of(uint32_t code) { return __uint_as_float(code & 0x80000000u ? (code == 0xffffffffu ? 0x7fc00000u : code & 0x7fffffffu) : ~code); }

__device__ __forceinline__ uint32_t wave_max(uint32_t v)
{
    v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x111, 0xf, 0xf, false));
    v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x112, 0xf, 0xf, false));
    v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x114, 0xf, 0xf, false));
    v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x118, 0xf, 0xf, false));
    v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x142, 0xa, 0xf, false));
    v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x143, 0xc, 0xf, false));
    return (uint32_t)__builtin_amdgcn_readlane((int)v, 63);
}
// Sum over the wave, in one order
__device__ __forceinline__ float wave_sum(float v)
{
    auto add = [&](float from) { v += from; };
    add(__int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x111, 0xf, 0xf, false)));
    add(__int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x112, 0xf, 0xf, false)));
    add(__int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x114, 0xf, 0xf, false)));
    add(__int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x118, 0xf, 0xf, false)));
    add(__int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x142, 0xa, 0xf, false)));
    add(__int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x143, 0xc, 0xf, false)));
    return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), 63));
}

struct RouteParams {
    const void *logits;
    float *weights;
    int *experts, *rows, *places, *offsets, *counts;  // counts: [workgroups][E], of more than one workgroup
    long ld;
    int M, E, k, each, normalize, workgroups;         // each: tokens of a workgroup
};

// Places of the rows of a workgroup's tokens: the rows of its experts begin at `base`.  Every wave has a run of tokens and counters of its own,
// [kWaves][E]; a token's experts differ, so its lanes count without meeting, and the waves' tokens are in order.
__device__ __forceinline__ void place_rows(const RouteParams &p, int token0, int token1, const int *base, int *counters)
{
    const int t = threadIdx.x, lane = t % 64, wave = t / 64, step = (token1 - token0 + kWaves - 1) / kWaves;
    const int mine0 = min(token0 + wave * step, token1), mine1 = min(mine0 + step, token1);
    int *const own = counters + wave * p.E;
    for (int i = t; i < kWaves * p.E; i += kThreads) counters[i] = 0;
    __syncthreads();
    for (long i = (long)mine0 * p.k + lane; i < (long)mine1 * p.k; i += 64) {
        const int e = p.experts[i];
        if (e >= 0) atomicAdd(own + e, 1);
    }
    __syncthreads();
    for (int e = t; e < p.E; e += kThreads) {
        int at = base[e];
        for (int w = 0; w < kWaves; w++) {
            const int n = counters[w * p.E + e];
            counters[w * p.E + e] = at;
            at += n;
        }
    }
    __syncthreads();
    const int per = 64 / p.k, turn = lane / p.k;  // tokens of one load; when it is this lane's turn
    for (int first = mine0; first < mine1; first += per) {
        const int token = first + turn;
        const bool here = turn < per && token < mine1;
        const long at = (long)first * p.k + lane;
        const int e = here ? p.experts[at] : -1;
        int place = -1;
        for (int s = 0; s < per && first + s < mine1; s++) {
            if (s == turn && e >= 0) {
                place = own[e];
                own[e] = place + 1;
            }
            asm volatile("" ::: "memory");  // one token after the other
            __builtin_amdgcn_wave_barrier();
        }
        if (here) {
            p.places[at] = place;
            if (place >= 0) p.rows[place] = token;
        }
    }
}

// Where the experts' rows begin, from their numbers: base of E (the numbers become the beginnings) and the number of all rows.  By the first wave.
__device__ __forceinline__ int begin_rows(int *numbers, int E, int lane)
{
    int before = 0;
    for (int first = 0; first < E; first += 64) {
        const int e = first + lane, n = e < E ? numbers[e] : 0, sum = wave_scan(n);
        if (e < E) numbers[e] = before + sum - n;
        before += __builtin_amdgcn_readlane(sum, 63);
    }
    return before;
}

// A wave takes a token at a time, lane l the experts l, l + 64 ..; a choice is one maximum over the wave and a vote.  V: experts a lane.  ONE: all tokens in
// this workgroup, which places their rows too.
template <int DTYPE, int V, bool ONE> __global__ __launch_bounds__(kThreads) void route_choose(const RouteParams p)
{
    using T = typename Element<DTYPE>::type;
    extern __shared__ __attribute__((aligned(16))) int shared[];  // E numbers, then (ONE) the waves' counters
    __shared__ int all_rows;
    const int t = threadIdx.x, lane = t % 64, wave = __builtin_amdgcn_readfirstlane(t / 64);
    const int token0 = (int)blockIdx.x * p.each, token1 = min(token0 + p.each, p.M);
    for (int e = t; e < p.E; e += kThreads) shared[e] = 0;
    __syncthreads();
    T next[V];
    auto load = [&](int token) {
        const T *const row = static_cast<const T *>(p.logits) + (long)token * p.ld;
#pragma unroll
        for (int i = 0; i < V; i++)
            if (i * 64 + lane < p.E) next[i] = row[i * 64 + lane];
    };
    if (token0 + wave < token1) load(token0 + wave);
    for (int token = token0 + wave; token < token1; token += kWaves) {
        float v[V];
        uint32_t code[V];
#pragma unroll
        for (int i = 0; i < V; i++) {
            v[i] = i * 64 + lane < p.E ? (float)next[i] : -__builtin_inff();
            code[i] = order_code(v[i]);
        }
        if (token + kWaves < token1) load(token + kWaves);
        int expert = -1;      // lane j: choice j
        float logit = 0.f, top = 0.f;
        for (int j = 0; j < p.k; j++) {
            uint32_t mine = code[0];
#pragma unroll
            for (int i = 1; i < V; i++) mine = max(mine, code[i]);
            const uint32_t best = wave_max(mine);
            if (best == 0) break;
            int e = -1;
#pragma unroll
            for (int i = 0; i < V; i++) {
                const uint64_t who = __ballot(code[i] == best);
                if (e < 0 && who) {
                    const int l = __builtin_ctzll(who);
                    e = i * 64 + l;
                    if (lane == l) code[i] = 0;
                }
            }
            if (j == 0) top = value_of(best);
            if (lane == j) expert = e, logit = value_of(best);
        }
        const bool open = expert >= 0;  // (of lanes past the choices too: no)
        const float part = open ? expf(logit - top) : 0.f;
        float whole;
        if (p.normalize) {
            whole = wave_sum(part);
        } else {
            float sum = 0.f;
#pragma unroll
            for (int i = 0; i < V; i++) sum += expf(v[i] - top);
            whole = wave_sum(sum);
        }
        if (lane < p.k) {
            const long at = (long)token * p.k + lane;
            p.weights[at] = open ? part / whole : 0.f;
            p.experts[at] = expert;
            if (open) atomicAdd(shared + expert, 1);
        }
    }
    __syncthreads();
    if constexpr (ONE) {
        if (wave == 0) {
            const int rows = begin_rows(shared, p.E, lane);
            if (lane == 0) all_rows = rows;
        }
        __syncthreads();
        for (int e = t; e <= p.E; e += kThreads) p.offsets[e] = e < p.E ? shared[e] : all_rows;
        for (int r = all_rows + t; r < p.M * p.k; r += kThreads) p.rows[r] = -1;
        place_rows(p, token0, token1, shared, shared + p.E);
    } else {
        for (int e = t; e < p.E; e += kThreads) p.counts[(long)blockIdx.x * p.E + e] = shared[e];
    }
}

// Places of all rows, from the numbers that every workgroup of route_choose left: each adds up for itself what is before it (256 rows of E numbers at
// the most, from L2), which saves a launch in between.
__global__ __launch_bounds__(kThreads) void route_place(const RouteParams p)
{
    extern __shared__ __attribute__((aligned(16))) int shared[];  // E beginnings, kThreads partial sums twice, then the waves' counters
    __shared__ int all_rows;
    int *const begin = shared, *const before = shared + p.E, *const whole = before + kThreads, *const counters = before;
    const int t = threadIdx.x, parts = kThreads / p.E, part = t / p.E, e = t - part * p.E;
    int sum = 0, mine = 0;
    if (part < parts)
        for (int g = part; g < p.workgroups; g += parts) {
            const int n = p.counts[(long)g * p.E + e];
            sum += n;
            if (g < (int)blockIdx.x) mine += n;
        }
    before[t] = mine, whole[t] = sum;
    __syncthreads();
    if (t < p.E) {
        for (int i = 1; i < parts; i++) mine += before[i * p.E + t], sum += whole[i * p.E + t];
        begin[t] = sum;
    }
    __syncthreads();
    if (t < 64) {
        const int rows = begin_rows(begin, p.E, t);
        if (t == 0) all_rows = rows;
    }
    __syncthreads();
    if (blockIdx.x == 0)
        for (int i = t; i <= p.E; i += kThreads) p.offsets[i] = i < p.E ? begin[i] : all_rows;
    __syncthreads();
    if (t < p.E) begin[t] += mine;
    __syncthreads();
    const int token0 = (int)blockIdx.x * p.each, token1 = min(token0 + p.each, p.M);
    // (unsigned: the step behind the last row may pass 2^31)
    for (uint32_t r = (uint32_t)max(all_rows, token0 * p.k) + t; r < (uint32_t)(token1 * p.k); r += kThreads) p.rows[r] = -1;
    place_rows(p, token0, token1, begin, counters);
}

struct RouteGradParams {
    const float *dweights, *weights;
    const int *experts;
    const void *logits;
    void *dlogits;
    long ld;
    int M, E, k, normalize;
};

// A wave takes a token; its choices' weights and gradients go from lane to lane
template <int DTYPE, int V> __global__ __launch_bounds__(256) void route_grad(const RouteGradParams p)
{
    using T = typename Element<DTYPE>::type;
    const int lane = threadIdx.x % 64, token = __builtin_amdgcn_readfirstlane((int)blockIdx.x * 4 + (int)threadIdx.x / 64);
    if (token >= p.M) return;
    const long at = (long)token * p.k + lane;
    const int expert = lane < p.k ? p.experts[at] : -1;
    const bool open = expert >= 0;
    const float w = open ? p.weights[at] : 0.f, g = open ? p.dweights[at] : 0.f, mean = wave_sum(w * g);
    float chosen[V], part[V];  // the gradient of the expert's weight; what the expert's softmax is
    if (p.normalize) {
#pragma unroll
        for (int i = 0; i < V; i++) chosen[i] = part[i] = 0.f;
    } else {
        const T *const row = static_cast<const T *>(p.logits) + (long)token * p.ld;
        uint32_t most = 0;
        float sum = 0.f;
#pragma unroll
        for (int i = 0; i < V; i++) {
            part[i] = i * 64 + lane < p.E ? (float)row[i * 64 + lane] : -__builtin_inff();
            most = max(most, order_code(part[i]));
            chosen[i] = 0.f;
        }
        most = wave_max(most);
        const float top = value_of(most);
#pragma unroll
        for (int i = 0; i < V; i++) {
            part[i] = most ? expf(part[i] - top) : 0.f;
            sum += part[i];
        }
        sum = wave_sum(sum);
#pragma unroll
        for (int i = 0; i < V; i++) part[i] = most ? part[i] / sum : 0.f;
    }
    for (int j = 0; j < p.k; j++) {
        const int e = __builtin_amdgcn_readlane(expert, j);
        if (e < 0) break;
        const float gj = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(g), j)), wj = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(w), j));
#pragma unroll
        for (int i = 0; i < V; i++)
            if (e == i * 64 + lane) {
                chosen[i] = gj;
                if (p.normalize) part[i] = wj;
            }
    }
    T *const out = static_cast<T *>(p.dlogits) + (long)token * p.E;
#pragma unroll
    for (int i = 0; i < V; i++)
        if (i * 64 + lane < p.E) out[i * 64 + lane] = (T)(part[i] * (chosen[i] - mean));
}

// One workgroup for few tokens; else at most 256, so that each can add the others' numbers up
constexpr int kOneMost = 128;
int tokens_each(int M) { return M <= kOneMost ? M : (M + 255) / 256 > kWaves ? (M + 255) / 256 : kWaves; }
int workgroups(int M) { return (int)(((long)M + tokens_each(M) - 1) / tokens_each(M)); }

template <int DTYPE, int V> hipError_t launch_v(const RouteParams &p, hipStream_t stream)
{
    const unsigned n = (unsigned)workgroups(p.M), numbers = (unsigned)p.E * 4, counters = numbers * kWaves;
    if (n == 1) {
        route_choose<DTYPE, V, true><<<1, kThreads, numbers + counters, stream>>>(p);
        return hipGetLastError();
    }
    route_choose<DTYPE, V, false><<<n, kThreads, numbers, stream>>>(p);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    route_place<<<n, kThreads, numbers + (counters > 8 * kThreads ? counters : 8 * kThreads), stream>>>(p);
    return hipGetLastError();
}
template <int DTYPE> hipError_t launch_choose(const RouteParams &p, hipStream_t stream)
{
    return p.E <= 64 ? launch_v<DTYPE, 1>(p, stream) : p.E <= 128 ? launch_v<DTYPE, 2>(p, stream) : p.E <= 256 ? launch_v<DTYPE, 4>(p, stream)
           : p.E <= 512 ? launch_v<DTYPE, 8>(p, stream) : launch_v<DTYPE, 16>(p, stream);
}

template <int DTYPE> hipError_t launch_grad(const RouteGradParams &p, hipStream_t stream)
{
    const unsigned n = (unsigned)(((long)p.M + 3) / 4);
    if (p.E <= 64) route_grad<DTYPE, 1><<<n, 256, 0, stream>>>(p);
    else if (p.E <= 128) route_grad<DTYPE, 2><<<n, 256, 0, stream>>>(p);
    else if (p.E <= 256) route_grad<DTYPE, 4><<<n, 256, 0, stream>>>(p);
    else if (p.E <= 512) route_grad<DTYPE, 8><<<n, 256, 0, stream>>>(p);
    else route_grad<DTYPE, 16><<<n, 256, 0, stream>>>(p);
    return hipGetLastError();
}

}  // namespace

size_t route_workspace(int M, int E, int) { return workgroups(M) == 1 ? 0 : ((size_t)workgroups(M) * (size_t)E * 4 + 15) / 16 * 16; }

hipError_t launch_route(int dtype, const RouteArgs &a, hipStream_t stream)
{
    const RouteParams p = {a.logits, a.weights, a.experts, a.rows, a.places, a.offsets, a.workspace, a.ld, a.M, a.E, a.k, tokens_each(a.M), a.normalize, workgroups(a.M)};
    return dtype == 0 ? launch_choose<0>(p, stream) : dtype == 1 ? launch_choose<1>(p, stream) : launch_choose<2>(p, stream);
}

hipError_t launch_route_grad(int dtype, const RouteGradArgs &a, hipStream_t stream)
{
    // a launch may hold 2^32 threads, 64 a token (a loop over tokens inside the kernel took 4-9 % longer)
    constexpr long kMost = 1l << 25;
    const long element = dtype == 0 ? 4 : 2;
    for (long first = 0; first < a.M; first += kMost) {
        const long M = a.M - first < kMost ? a.M - first : kMost, choice = first * a.k;
        const RouteGradParams p = {a.dweights + choice, a.weights + choice, a.experts + choice, static_cast<const char *>(a.logits) + first * a.ld * element,
                                   static_cast<char *>(a.dlogits) + first * a.E * element, a.ld, (int)M, a.E, a.k, a.normalize};
        const hipError_t e = dtype == 0 ? launch_grad<0>(p, stream) : dtype == 1 ? launch_grad<1>(p, stream) : launch_grad<2>(p, stream);
        if (e != hipSuccess) return e;
    }
    return hipSuccess;
}

}  // namespace tab
