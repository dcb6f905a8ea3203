// moe_route.hip -- the experts of each token and their weights.
//
// A wave takes a token, a lane V neighbouring experts, so that of equal scores
// the lowest lane's lowest is the first.  Scores are held as integers that
// compare as they do (NaN first, hidden experts last); the best is found by
// exchanges among lanes, k times.
//
// The order is that of f64 scores.  Where a score is the logit itself f32 holds
// it.  Else f32 scores are tried: their errors are below SURE, so two that are
// further apart have the right order, and only a token of which some that matter
// are not is done again in f64 (a few in a thousand), and so is one whose scores
// leave the range of f32.
//
// Bound by the issue of instructions, 670 vector and 350 scalar ones a token of
// 256 experts in groups: 8192 such tokens take 14.4 us, where their logits could
// be read in 1.8, 61 tokens 5.4; one of 128 experts 3.4.  Several tokens a wave,
// one after the other, took longer.
#include <hip/hip_runtime.h>
#include <math.h>

#include <type_traits>

#include "../../include/ggml_hip_moe.h"

namespace {

constexpr int WAVES = 4;

struct RouteArgs {
    const float *logits, *bias;
    int64_t logits_stride, ids_stride, weights_stride;
    int32_t *ids;
    float *weights;
    int n_tokens, n_experts, gating, n_groups, n_keep, group_top, k, renormalize;
    float min_sum, scale;
};

// Scores as integers of the same order.
template <typename S>
struct Key;

template <>
struct Key<float> {
    typedef int T;
    static constexpr T HIDDEN = (int)(1u << 31), NAN_FIRST = 0x7fffffff;
    static __device__ __forceinline__ T bits(float s) { return __float_as_int(s); }
    static __device__ __forceinline__ float from(T b) { return __int_as_float(b); }
};

template <>
struct Key<double> {
    typedef long long T;
    static constexpr T HIDDEN = (long long)(1ull << 63), NAN_FIRST = 0x7fffffffffffffffll;
    static __device__ __forceinline__ T bits(double s) { return __double_as_longlong(s); }
    static __device__ __forceinline__ double from(T b) { return __longlong_as_double(b); }
};

// -infinity is HIDDEN.
template <typename S>
__device__ __forceinline__ typename Key<S>::T key_of(S s) {
    typedef typename Key<S>::T T;
    const T b = Key<S>::bits(s + (S)0);  // -0 is 0
    const T k = b ^ ((b >> (8 * sizeof(T) - 1)) & Key<S>::NAN_FIRST);
    return s != s ? Key<S>::NAN_FIRST : s == -(S)INFINITY ? Key<S>::HIDDEN : k;
}

template <typename S>
__device__ __forceinline__ S score_of(typename Key<S>::T k) {
    return k == Key<S>::NAN_FIRST ? (S)NAN : Key<S>::from(k ^ ((k >> (8 * sizeof(k) - 1)) & Key<S>::NAN_FIRST));
}

// Two values, the lane's own and that of a lane that differs in bit STEP of its number, in either order, if lanes that
// agree in the higher bits have the same value.
typedef uint32_t v2u __attribute__((ext_vector_type(2)));
template <int STEP>
__device__ __forceinline__ void pair(int x, int &y, int &z) {
    if constexpr (STEP < 4) {
        // quad_perm 1 0 3 2, quad_perm 2 3 0 1, row_half_mirror, row_mirror
        constexpr int CONTROL[4] = {0xB1, 0x4E, 0x141, 0x140};
        y = x;
        z = __builtin_amdgcn_update_dpp(x, x, CONTROL[STEP], 0xf, 0xf, false);
    } else {
        const v2u r = STEP == 4 ? __builtin_amdgcn_permlane16_swap(x, x, false, false) : __builtin_amdgcn_permlane32_swap(x, x, false, false);
        y = (int)r.x, z = (int)r.y;
    }
}
template <int STEP>
__device__ __forceinline__ void pair(long long x, long long &y, long long &z) {
    int ly, lz, hy, hz;
    pair<STEP>((int)x, ly, lz);
    pair<STEP>((int)(x >> 32), hy, hz);
    y = (long long)((unsigned long long)(uint32_t)hy << 32 | (uint32_t)ly);
    z = (long long)((unsigned long long)(uint32_t)hz << 32 | (uint32_t)lz);
}
template <int STEP>
__device__ __forceinline__ void pair(float x, float &y, float &z) {
    int iy, iz;
    pair<STEP>(__float_as_int(x), iy, iz);
    y = __int_as_float(iy), z = __int_as_float(iz);
}
template <int STEP>
__device__ __forceinline__ void pair(double x, double &y, double &z) {
    long long iy, iz;
    pair<STEP>(__double_as_longlong(x), iy, iz);
    y = __longlong_as_double(iy), z = __longlong_as_double(iz);
}

// f (commutative) over the lanes of 2^STEPS neighbours, in all of them.
template <int STEP, int STEPS, typename T, typename F>
__device__ __forceinline__ T over(T x, F f) {
    if constexpr (STEP == STEPS) {
        return x;
    } else {
        T y, z;
        pair<STEP>(x, y, z);
        return over<STEP + 1, STEPS>(f(y, z), f);
    }
}
template <typename T>
__device__ __forceinline__ T largest(T x) {
    return over<0, 6>(x, [](T a, T b) { return a > b ? a : b; });
}
// A lane's value; the lane is the same for all.
__device__ __forceinline__ int lane_value(int x, int lane) { return __builtin_amdgcn_readlane(x, lane); }
__device__ __forceinline__ long long lane_value(long long x, int lane) {
    const uint32_t lo = (uint32_t)lane_value((int)x, lane), hi = (uint32_t)lane_value((int)(x >> 32), lane);
    return (long long)((unsigned long long)hi << 32 | lo);
}

// The largest key, the same for all lanes.
__device__ __forceinline__ int best_of(int x) {
    // Towards lane 63: rows of 16 by shifts, then the rows' last lanes forward.
    constexpr int LOW = (int)(1u << 31);
    x = max(x, __builtin_amdgcn_update_dpp(LOW, x, 0x111, 0xf, 0xf, false));
    x = max(x, __builtin_amdgcn_update_dpp(LOW, x, 0x112, 0xf, 0xf, false));
    x = max(x, __builtin_amdgcn_update_dpp(LOW, x, 0x114, 0xf, 0xf, false));
    x = max(x, __builtin_amdgcn_update_dpp(LOW, x, 0x118, 0xf, 0xf, false));
    x = max(x, __builtin_amdgcn_update_dpp(LOW, x, 0x142, 0xa, 0xf, false));
    x = max(x, __builtin_amdgcn_update_dpp(LOW, x, 0x143, 0xc, 0xf, false));
    return lane_value(x, 63);
}
__device__ __forceinline__ long long best_of(long long x) { return lane_value(largest(x), 0); }

__device__ __forceinline__ double exponential(double x) { return exp(x); }
__device__ __forceinline__ float exponential(float x) { return __builtin_amdgcn_exp2f(x * 1.44269504f); }
__device__ __forceinline__ double inverse(double x) { return 1.0 / x; }
__device__ __forceinline__ float inverse(float x) { return __builtin_amdgcn_rcpf(x); }

// Two f32 scores that differ by more than SURE times the larger of 1 and their size have the order of the exact ones.
// p is below 1 and off by the exponential (its argument's rounding, |l| 2^-24 relative, matters as x e^-x does, and its
// own, 2^-23), the sum of at most 1024 (sums of 16 and then 6 more levels, 22 * 2^-24) and the reciprocal (2^-23): under
// 2^-19; adding the bias is off by half a step of the sum, 2^-24 of its size.
//
// A group's score is the sum of two of them and off by what both are and by half a step of its own.  Its two may be
// large and of opposite signs, and it then small: its error goes by their size, not by its own.  With the larger of 1 and
// their magnitudes as a unit it is below 2 * 2^-19 (p) + 2 * 2^-24 (biases) + 2 * 2^-24 (sum), little over half of SURE.
// So a group comes before another for sure if its score less SURE units is above the other's and SURE of its own (whose
// roundings are 2 * 2^-24 each).
constexpr float SURE = 0x1p-17f;

template <typename S>
__device__ __forceinline__ bool apart(S a, S b) {
    return a - b > SURE * fmaxf(1.0f, fmaxf(fabsf((float)a), fabsf((float)b)));
}

// The softmax's maximum and sum.
template <typename S>
struct Softmax {
    S top, sum;
};

template <typename S>
__device__ __forceinline__ S p_of(const RouteArgs &a, const Softmax<S> &m, float l) {
    if (a.gating == HIP_QMM_ROUTE_SOFTMAX) return exponential((S)l - m.top) * inverse(m.sum);
    if (a.gating == HIP_QMM_ROUTE_SIGMOID) return inverse((S)1 + exponential(-(S)l));
    return (S)l;
}

template <typename S, int V>
__device__ __forceinline__ Softmax<S> softmax_of(const float (&l)[V]) {
    float m = l[0];
    bool bad = false;
#pragma unroll
    for (int v = 0; v < V; ++v) {
        m = fmaxf(m, l[v]);
        bad |= l[v] != l[v];
    }
    m = largest(m);
    const S top = __any(bad) ? (S)NAN : (S)m;
    S sum = 0;
#pragma unroll
    for (int v = 0; v < V; ++v)
        if (l[v] != -INFINITY) sum += exponential((S)l[v] - top);
    return {top, over<0, 6>(sum, [](S a, S b) { return a + b; })};
}

// Lane j's id: the j-th best.  False: f32 scores do not tell.
template <typename S, int V, bool EXACT>
__device__ __forceinline__ bool choose(const RouteArgs &a, const float (&l)[V], const float (&b)[V], void *shared, int &id) {
    typedef typename Key<S>::T T;
    const int lane = threadIdx.x & 63;
    const bool sums = a.n_groups > a.n_keep && a.group_top > 1;
    Softmax<S> m = {0, 1};
    if (a.gating == HIP_QMM_ROUTE_SOFTMAX && (a.bias || sums)) m = softmax_of<S>(l);
    T key[V];
    bool finite = true;
#pragma unroll
    for (int v = 0; v < V; ++v) {
        const bool hidden = l[v] == -INFINITY || b[v] == -INFINITY;
        const S s = a.bias ? p_of(a, m, l[v]) + (S)b[v] : (S)l[v];
        if constexpr (!EXACT) {
            finite &= hidden || s - s == 0;
            const T b = Key<S>::bits(s + (S)0);
            key[v] = hidden ? Key<S>::HIDDEN : b ^ ((b >> 31) & Key<S>::NAN_FIRST);
        } else {
            key[v] = hidden ? Key<S>::HIDDEN : key_of<S>(s);
        }
    }
    if (!EXACT && !__all(finite)) return false;
    bool sure = true;
    if (a.n_groups > a.n_keep) {
        const int size = a.n_experts / a.n_groups;
        auto take = [](T &first, T &second, T x, T y) {  // the two best of first >= second and x >= y
            const T low = first < x ? first : x, next = second > y ? second : y;
            first = first > x ? first : x;
            second = low > next ? low : next;
        };
        T first = Key<S>::HIDDEN, second = Key<S>::HIDDEN;
        const int lanes = size / V;
        int group = lane, at = 1;  // the group whose score a lane has, and the lanes from one to the next
        const bool aligned = size % V == 0 && (lanes & (lanes - 1)) == 0;  // groups of 2^n whole lanes
        if (aligned) {
#pragma unroll
            for (int v = 0; v < V; ++v) take(first, second, key[v], Key<S>::HIDDEN);
            auto merge = [&](auto step) {
                constexpr int STEP = decltype(step)::value;
                T x, y;
                pair<STEP>(first, first, x);
                pair<STEP>(second, second, y);
                take(first, second, x, y);
            };
            if (lanes > 1) merge(std::integral_constant<int, 0>());
            if (lanes > 2) merge(std::integral_constant<int, 1>());
            if (lanes > 4) merge(std::integral_constant<int, 2>());
            if (lanes > 8) merge(std::integral_constant<int, 3>());
            if (lanes > 16) merge(std::integral_constant<int, 4>());
            if (lanes > 32) merge(std::integral_constant<int, 5>());
            group = lane / lanes;
            at = lanes;
        } else {
            T *keys = reinterpret_cast<T *>(shared);
#pragma unroll
            for (int v = 0; v < V; ++v) keys[lane * V + v] = key[v];
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            __builtin_amdgcn_wave_barrier();
            if (lane < a.n_groups)
                for (int i = 0; i < size; ++i) take(first, second, keys[lane * size + i], Key<S>::HIDDEN);
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            __builtin_amdgcn_wave_barrier();
        }
        T mine = first;
        float unit = 1.0f;  // of f32 scores' errors
        if (first != Key<S>::HIDDEN) {
            S x = score_of<S>(first), y = 0;
            if (sums) {
                if (second != Key<S>::HIDDEN) y = score_of<S>(second);
                if (!a.bias) x = p_of(a, m, (float)x), y = second != Key<S>::HIDDEN ? p_of(a, m, (float)y) : y;
                mine = key_of<S>(x + y);
                sure = x + y - (x + y) == 0;  // else beyond f32: below it not to be taken for hidden
            }
            unit = fmaxf(1.0f, fmaxf(fabsf((float)x), fabsf((float)y)));
        }
        if (group >= a.n_groups) mine = Key<S>::HIDDEN;
        int before = 0;  // groups that come before this lane's
        for (int g = 0; g < a.n_groups; ++g) {
            const T x = lane_value(mine, g * at);
            before += x > mine || (x == mine && g < group);
        }
        const bool kept = group < a.n_groups && before < a.n_keep;
        if constexpr (!EXACT) {
            // The worst that is kept at its lowest, and the best that is not at its highest.
            const float score = score_of<S>(mine), reach = SURE * unit;
            const T end = mine == Key<S>::HIDDEN ? mine : key_of<S>(kept ? score - reach : score + reach);
            const T out = largest(kept ? Key<S>::HIDDEN : end), in = ~largest(kept ? ~end : Key<S>::HIDDEN);
            sure = __all(sure) && (out == Key<S>::HIDDEN || in > out);
        }
        if (aligned) {
#pragma unroll
            for (int v = 0; v < V; ++v) key[v] = kept ? key[v] : Key<S>::HIDDEN;
        } else {
            const unsigned long long who = __ballot(kept);
#pragma unroll
            for (int v = 0; v < V; ++v) {
                const int e = lane * V + v;
                if (e >= a.n_experts || !((who >> (e / size)) & 1)) key[v] = Key<S>::HIDDEN;
            }
        }
    }
    id = -1;
    T mine = Key<S>::HIDDEN;  // of the lane's id; in lane k of the one that would be next
    // The lane's keys in descending order, of equal ones the lower expert's first, and which they are, four bits each: a
    // round then looks at one key a lane (8192 tokens, 8 of 256 in groups, 17.0 -> 15.3 us; 8 of 512 16.5 -> 15.9, 1 of 512
    // 11.9 -> 13.0).  Of 16 keys the sort would cost more.
    constexpr bool SORTED = V <= 8;
    uint32_t order = 0;
    if constexpr (SORTED) {
        int at[V];
#pragma unroll
        for (int v = 0; v < V; ++v) at[v] = v;
#pragma unroll
        for (int pass = 0; pass < V; ++pass)
#pragma unroll
            for (int v = pass & 1; v + 1 < V; v += 2) {
                const bool swap = key[v + 1] > key[v];
                const T x = key[v], y = key[v + 1];
                const int i = at[v], j = at[v + 1];
                key[v] = swap ? y : x, key[v + 1] = swap ? x : y;
                at[v] = swap ? j : i, at[v + 1] = swap ? i : j;
            }
#pragma unroll
        for (int v = 0; v < V; ++v) order |= (uint32_t)at[v] << (4 * v);
    }
    for (int j = 0; j < a.k + (EXACT ? 0 : 1); ++j) {
        T best = key[0];
        if constexpr (!SORTED) {
#pragma unroll
            for (int v = 1; v < V; ++v) best = key[v] > best ? key[v] : best;
        }
        const T here = best;
        best = best_of(best);
        if (best == Key<S>::HIDDEN) break;
        if (lane == j) mine = best;
        if (!EXACT && j == a.k) break;
        const int owner = __ffsll((long long)__ballot(here == best)) - 1;
        int v_of;
        if constexpr (SORTED) {
            v_of = lane_value((int)order, owner) & 15;
            if (lane == owner) {
#pragma unroll
                for (int v = 0; v + 1 < V; ++v) key[v] = key[v + 1];
                key[V - 1] = Key<S>::HIDDEN;
                order >>= 4;
            }
        } else {
            int at = V;  // the lane's first expert with that score
#pragma unroll
            for (int v = V - 1; v >= 0; --v) at = key[v] == best ? v : at;
            v_of = lane_value(at, owner);
#pragma unroll
            for (int v = 0; v < V; ++v) key[v] = lane == owner && v == v_of ? Key<S>::HIDDEN : key[v];
        }
        if (lane == j) id = owner * V + v_of;
    }
    if constexpr (!EXACT) {
        // Each from the next, if there is one.  (Of 64 the last is not compared with a 65th.)
        const int next = __shfl_down(mine, 1);
        const bool two = lane < a.k && lane < 63 && mine != Key<S>::HIDDEN && next != Key<S>::HIDDEN;
        if (__any(two && !apart(score_of<S>(mine), score_of<S>(next))) || a.k == 64) sure = false;
    }
    return sure;
}

// V logits of a token, those of experts that are not there -infinity.
template <int V>
__device__ __forceinline__ void load(const float *row, int n, float none, float (&x)[V]) {
    const int lane = threadIdx.x & 63;
    constexpr int W = V < 4 ? V : 4;  // values of a load
    typedef float vec __attribute__((ext_vector_type(W), aligned(4)));
    if (V > 1 && n % V == 0) {
#pragma unroll
        for (int v = 0; v < V; v += W) {
            vec u = none;
            if (lane * V < n) u = *reinterpret_cast<const vec *>(row + lane * V + v);
#pragma unroll
            for (int i = 0; i < W; ++i) x[v + i] = u[i];
        }
    } else {
#pragma unroll
        for (int v = 0; v < V; ++v) x[v] = lane * V + v < n ? row[lane * V + v] : none;
    }
}

template <int V>
__global__ __launch_bounds__(64 * WAVES) void route_kernel(RouteArgs a) {
    __shared__ double shared[WAVES][V * 64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int t = blockIdx.x * WAVES + wave;
    if (t >= a.n_tokens) return;
    const float *row = a.logits + (int64_t)t * a.logits_stride;
    float l[V], b[V];
#pragma unroll
    for (int v = 0; v < V; ++v) b[v] = 0.0f;
    load<V>(row, a.n_experts, -INFINITY, l);
    if (a.bias) load<V>(a.bias, a.n_experts, 0.0f, b);
    int id;
    const bool logits = !a.bias && (a.n_groups == a.n_keep || a.group_top == 1);  // all that is compared
    if (logits)
        choose<float, V, true>(a, l, b, shared[wave], id);
    else if (!choose<float, V, false>(a, l, b, shared[wave], id))
        choose<double, V, true>(a, l, b, shared[wave], id);

    // The weights, in f64 throughout, in lanes 0 .. k - 1.
    auto chosen = [&](auto x, auto f) { return a.k <= 8 ? over<0, 3>(x, f) : a.k <= 16 ? over<0, 4>(x, f) : over<0, 6>(x, f); };
    auto add = [](double x, double y) { return x + y; };
    double w = 0.0;
    const float x = id >= 0 ? row[id] : -INFINITY;
    if (a.gating == HIP_QMM_ROUTE_SOFTMAX_CHOSEN) {
        // The largest, or NaN if one is.
        const float top = chosen(x, [](float x, float y) { return x != x || x > y ? x : y; });
        if (id >= 0) w = exp((double)x - (double)top);
        w /= chosen(w, add);
    } else {
        Softmax<double> m = {0.0, 1.0};
        if (a.gating == HIP_QMM_ROUTE_SOFTMAX) m = softmax_of<double>(l);
        if (id >= 0) w = p_of(a, m, x);
    }
    if (id < 0) w = 0.0;
    if (a.renormalize) {
        const double sum = chosen(w, add);
        w /= sum < (double)a.min_sum ? (double)a.min_sum : sum;
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
    if (!logits || !ids || !weights || ((uintptr_t)logits | (uintptr_t)bias | (uintptr_t)ids | (uintptr_t)weights) % 4 ||
        logits_stride < n_experts || ids_stride < k || weights_stride < k ||
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
