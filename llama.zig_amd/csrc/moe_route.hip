// moe_route.hip -- the experts of each token and their weights.
//
// A wave takes a token; expert v*64 + lane is its lane's v-th.  Scores are f64,
// held as 64-bit keys whose integer order is the scores' (NaN first, hidden
// experts last), so every comparison is exact and one for all cases.
#include <hip/hip_runtime.h>
#include <math.h>

#include "../../include/ggml_hip_moe.h"

namespace {

constexpr int WAVES = 4;
constexpr long long HIDDEN = (long long)(1ull << 63);

struct RouteArgs {
    const float *logits, *bias;
    int64_t logits_stride, ids_stride, weights_stride;
    int32_t *ids;
    float *weights;
    int n_tokens, n_experts, gating, n_groups, n_keep, group_top, k, renormalize;
    float min_sum, scale;
};

// f64 to an integer of the same order; NaN above all, -infinity HIDDEN.
__device__ __forceinline__ long long key_of(double s) {
    if (s != s) return 0x7fffffffffffffffll;
    if (s == -INFINITY) return HIDDEN;
    const long long b = __double_as_longlong(s + 0.0);  // -0 is 0
    return b ^ ((b >> 63) & 0x7fffffffffffffffll);
}

__device__ __forceinline__ double value_of(long long k) {
    return k == 0x7fffffffffffffffll ? (double)NAN : __longlong_as_double(k ^ ((k >> 63) & 0x7fffffffffffffffll));
}

__device__ __forceinline__ double wave_sum(double x) {
#pragma unroll
    for (int d = 32; d; d >>= 1) x += __shfl_xor(x, d);
    return x;
}

__device__ __forceinline__ double sigmoid(double x) { return 1.0 / (1.0 + exp(-x)); }

template <int V>
__global__ __launch_bounds__(64 * WAVES) void route_kernel(RouteArgs a) {
    __shared__ long long shared[WAVES][V * 64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int t = blockIdx.x * WAVES + wave;
    if (t >= a.n_tokens) return;
    const float *row = a.logits + (int64_t)t * a.logits_stride;
    float l[V];
#pragma unroll
    for (int v = 0; v < V; ++v) l[v] = v * 64 + lane < a.n_experts ? row[v * 64 + lane] : -INFINITY;

    // The softmax's maximum and sum.
    const bool softmax = a.gating == HIP_QMM_ROUTE_SOFTMAX;
    double top = 0.0, sum = 1.0;
    if (softmax) {
        float m = l[0];
        bool bad = false;
#pragma unroll
        for (int v = 0; v < V; ++v) {
            m = fmaxf(m, l[v]);
            bad |= l[v] != l[v];
        }
#pragma unroll
        for (int d = 32; d; d >>= 1) m = fmaxf(m, __shfl_xor(m, d));
        top = __any(bad) ? (double)NAN : (double)m;
        sum = 0.0;
#pragma unroll
        for (int v = 0; v < V; ++v)
            if (l[v] != -INFINITY) sum += exp((double)l[v] - top);
        sum = wave_sum(sum);
    }
    auto p_of = [&](float x) {
        return softmax ? exp((double)x - top) / sum : a.gating == HIP_QMM_ROUTE_SIGMOID ? sigmoid(x) : (double)x;
    };

    // Scores.  Without a bias the logits have their order; with groups of two best scores their sums are needed.
    const bool sums = a.n_groups > 1 && a.group_top > 1;
    long long key[V];
#pragma unroll
    for (int v = 0; v < V; ++v) {
        const int e = v * 64 + lane;
        key[v] = HIDDEN;
        if (e < a.n_experts && l[v] != -INFINITY) {
            const double b = a.bias ? (double)a.bias[e] : 0.0;
            if (b != -INFINITY) key[v] = key_of(a.bias ? p_of(l[v]) + b : (double)l[v]);
        }
    }
    if (a.n_groups > 1) {
        const int size = a.n_experts / a.n_groups;
#pragma unroll
        for (int v = 0; v < V; ++v) shared[wave][v * 64 + lane] = key[v];
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
        long long mine = HIDDEN;
        if (lane < a.n_groups) {
            long long first = HIDDEN, second = HIDDEN;
            for (int i = 0; i < size; ++i) {
                const long long k = shared[wave][lane * size + i];
                second = max(second, min(first, k));
                first = max(first, k);
            }
            mine = first;
            if (sums && first != HIDDEN) {
                double x = value_of(first), y = value_of(second);
                if (!a.bias) x = p_of((float)x), y = p_of((float)y);
                mine = key_of(second != HIDDEN ? x + y : x);
            }
        }
        int before = 0;  // groups that come before this lane's
        for (int g = 0; g < a.n_groups; ++g) {
            const long long other = __shfl(mine, g);
            before += other > mine || (other == mine && g < lane);
        }
        const unsigned long long kept = __ballot(lane < a.n_groups && before < a.n_keep);
#pragma unroll
        for (int v = 0; v < V; ++v) {
            const int e = v * 64 + lane;
            if (e >= a.n_experts || !((kept >> (e / size)) & 1)) key[v] = HIDDEN;
        }
    }

    // The k best, one after another; lane j keeps the j-th.
    int id = -1;
    for (int j = 0; j < a.k; ++j) {
        long long best = key[0];
        int at = lane;
#pragma unroll
        for (int v = 1; v < V; ++v)
            if (key[v] > best) best = key[v], at = v * 64 + lane;
#pragma unroll
        for (int d = 32; d; d >>= 1) {
            const long long b = __shfl_xor(best, d);
            const int i = __shfl_xor(at, d);
            if (b > best || (b == best && i < at)) best = b, at = i;
        }
        if (best == HIDDEN) break;
#pragma unroll
        for (int v = 0; v < V; ++v)
            if (at == v * 64 + lane) key[v] = HIDDEN;
        if (lane == j) id = at;
    }

    double w = 0.0;
    if (a.gating == HIP_QMM_ROUTE_SOFTMAX_CHOSEN) {
        const double x = id >= 0 ? (double)row[id] : -INFINITY;
        double m = x;
        const bool bad = __any(x != x);
#pragma unroll
        for (int d = 32; d; d >>= 1) m = fmax(m, __shfl_xor(m, d));
        if (bad) m = NAN;
        if (id >= 0) w = exp(x - m);
        w /= wave_sum(w);
    } else if (id >= 0) {
        w = p_of(row[id]);
    }
    if (id < 0) w = 0.0;
    if (a.renormalize) {
        const double total = wave_sum(w);
        w /= total < (double)a.min_sum ? (double)a.min_sum : total;
        if (id < 0) w = 0.0;
    }
    if (lane < a.k) {
        a.ids[(int64_t)t * a.ids_stride + lane] = id;
        a.weights[(int64_t)t * a.weights_stride + lane] = id < 0 ? 0.0f : (float)(w * (double)a.scale);
    }
}

}  // namespace

extern "C" int hip_qmm_moe_route(const float *logits, int64_t n_tokens, int64_t n_experts, int64_t logits_stride,
                                 const float *bias, int gating, int64_t n_groups, int64_t n_keep, int group_top,
                                 int64_t k, int renormalize, float min_sum, float scale, int32_t *ids,
                                 int64_t ids_stride, float *weights, int64_t weights_stride, void *stream) {
    const int64_t lim = (int64_t)1 << 40;
    if (n_tokens < 0 || n_tokens > (1 << 24) || n_experts < 1 || n_experts > 1024 || gating < 0 || gating > 2 ||
        k < 1 || k > 64 || k > n_experts || n_groups < 1 || n_groups > 64 || n_experts % n_groups || n_keep < 1 ||
        n_keep > n_groups || group_top < 1 || group_top > 2 || !(min_sum >= 0.0f) || !isfinite(min_sum) ||
        !isfinite(scale))
        return (int)hipErrorInvalidValue;
    if (n_tokens == 0) return 0;
    if (!logits || !ids || !weights || logits_stride < n_experts || ids_stride < k || weights_stride < k ||
        logits_stride > lim || ids_stride > lim || weights_stride > lim)
        return (int)hipErrorInvalidValue;
    const RouteArgs a = {logits, bias, logits_stride, ids_stride, weights_stride, ids, weights, (int)n_tokens,
                         (int)n_experts, gating, (int)n_groups, (int)n_keep, group_top, (int)k, renormalize, min_sum,
                         scale};
    const dim3 grid((unsigned)((n_tokens + WAVES - 1) / WAVES)), block(64 * WAVES);
    hipStream_t s = (hipStream_t)stream;
    if (n_experts <= 64)
        hipLaunchKernelGGL(route_kernel<1>, grid, block, 0, s, a);
    else if (n_experts <= 128)
        hipLaunchKernelGGL(route_kernel<2>, grid, block, 0, s, a);
    else if (n_experts <= 256)
        hipLaunchKernelGGL(route_kernel<4>, grid, block, 0, s, a);
    else if (n_experts <= 512)
        hipLaunchKernelGGL(route_kernel<8>, grid, block, 0, s, a);
    else
        hipLaunchKernelGGL(route_kernel<16>, grid, block, 0, s, a);
    return (int)hipGetLastError();
}
