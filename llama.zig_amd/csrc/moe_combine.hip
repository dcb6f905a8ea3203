// moe_combine.hip -- the weighted sum of each token's experts' rows.  HBM bound,
// so the sums are in f64, which costs nothing, and rounded once: 4096 tokens of 8
// rows of 2048 take 57 us (5.3 TB/s, a copy's rate).
#include <hip/hip_runtime.h>

#include <algorithm>

#include "../../include/ggml_hip_moe.h"

namespace {

constexpr int THREADS = 256;

struct CombineArgs {
    const float *y, *weights, *add;
    const int32_t *ids;
    float *dst;
    int64_t y_token, y_row, weights_stride, ids_stride, add_stride, dst_stride;
    int64_t n_tokens, nrows;
    int n_ids;
};

// Four values of a row per thread, or the up to three that it ends with.  Rows need not be aligned to more than a value: a
// load or store of 16 bytes need not be (1789 tokens of 4 rows of 5174: 38 us, by single values 61).
typedef float vec __attribute__((ext_vector_type(4), aligned(4)));

template <int N>
__device__ __forceinline__ void combine(const CombineArgs &a, int64_t t, int64_t u) {
    double sum[N];
    auto load = [](const float *p, float (&v)[N]) {
        if constexpr (N == 4) {
            const vec x = *reinterpret_cast<const vec *>(p);
#pragma unroll
            for (int e = 0; e < N; ++e) v[e] = x[e];
        } else {
            v[0] = *p;
        }
    };
    float v[N];
#pragma unroll
    for (int e = 0; e < N; ++e) sum[e] = 0.0;
    if (a.add) {
        load(a.add + t * a.add_stride + u, v);
#pragma unroll
        for (int e = 0; e < N; ++e) sum[e] = v[e];
    }
    const float *y = a.y + t * a.y_token + u;
    for (int s = 0; s < a.n_ids; ++s) {
        if (a.ids && a.ids[t * a.ids_stride + s] < 0) continue;
        load(y + s * a.y_row, v);
        const double w = a.weights[t * a.weights_stride + s];
#pragma unroll
        for (int e = 0; e < N; ++e) sum[e] = fma(w, (double)v[e], sum[e]);
    }
    float *out = a.dst + t * a.dst_stride + u;
    if constexpr (N == 4)
        *reinterpret_cast<vec *>(out) = (vec){(float)sum[0], (float)sum[1], (float)sum[2], (float)sum[3]};
    else
        *out = (float)sum[0];
}

__global__ __launch_bounds__(THREADS) void combine_kernel(CombineArgs a) {
    const int64_t units = (a.nrows + 3) / 4, total = units * a.n_tokens, step = (int64_t)gridDim.x * THREADS;
    for (int64_t i = (int64_t)blockIdx.x * THREADS + threadIdx.x; i < total; i += step) {
        const int64_t t = i / units, u = (i - t * units) * 4;
        if (u + 4 <= a.nrows)
            combine<4>(a, t, u);
        else
            for (int64_t e = u; e < a.nrows; ++e) combine<1>(a, t, e);
    }
}

}  // namespace

extern "C" int hip_qmm_moe_combine(const float *y, int64_t n_tokens, int64_t n_ids, int64_t nrows,
                                   int64_t y_token_stride, int64_t y_row_stride, const float *weights,
                                   int64_t weights_stride, const int32_t *ids, int64_t ids_stride, const float *add,
                                   int64_t add_stride, float *dst, int64_t dst_stride, void *stream) {
    const int64_t lim = (int64_t)1 << 40;
    if (n_tokens < 0 || n_tokens > INT32_MAX || n_ids < 0 || n_ids > 65535 || nrows < 0 || nrows > INT32_MAX)
        return (int)hipErrorInvalidValue;
    if (n_tokens == 0 || nrows == 0) return 0;
    if (((uintptr_t)y | (uintptr_t)weights | (uintptr_t)ids | (uintptr_t)add | (uintptr_t)dst) % 4)
        return (int)hipErrorInvalidValue;
    if (!dst || dst_stride < nrows || dst_stride > lim || (add && (add_stride < nrows || add_stride > lim)))
        return (int)hipErrorInvalidValue;
    if (n_ids > 0 && (!y || !weights || y_token_stride < 0 || y_row_stride < 0 || y_token_stride > lim ||
                      y_row_stride > lim || weights_stride < n_ids || weights_stride > lim ||
                      (ids && (ids_stride < n_ids || ids_stride > lim))))
        return (int)hipErrorInvalidValue;
    if (add == dst && add_stride != dst_stride) return (int)hipErrorInvalidValue;
    const CombineArgs a = {y, weights, add, ids, dst, y_token_stride, y_row_stride, weights_stride, ids_stride,
                           add_stride, dst_stride, n_tokens, nrows, (int)n_ids};
    const int64_t units = n_tokens * ((nrows + 3) / 4);
    hipLaunchKernelGGL(combine_kernel, dim3((unsigned)std::min((units + THREADS - 1) / THREADS, (int64_t)1 << 20)),
                       dim3(THREADS), 0, (hipStream_t)stream, a);
    return (int)hipGetLastError();
}
