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

// N values of a row per thread; a row of threads covers a token's units.
template <int N>
__global__ __launch_bounds__(THREADS) void combine_kernel(CombineArgs a) {
    const int64_t units = a.nrows / N, total = units * a.n_tokens, step = (int64_t)gridDim.x * THREADS;
    for (int64_t i = (int64_t)blockIdx.x * THREADS + threadIdx.x; i < total; i += step) {
        const int64_t t = i / units, u = (i - t * units) * N;
        typedef float vec __attribute__((ext_vector_type(N)));
        double sum[N];
#pragma unroll
        for (int e = 0; e < N; ++e) sum[e] = 0.0;
        if (a.add) {
            const vec v = *reinterpret_cast<const vec *>(a.add + t * a.add_stride + u);
#pragma unroll
            for (int e = 0; e < N; ++e) sum[e] = v[e];
        }
        const float *y = a.y + t * a.y_token + u;
        for (int s = 0; s < a.n_ids; ++s) {
            if (a.ids && a.ids[t * a.ids_stride + s] < 0) continue;
            const vec v = *reinterpret_cast<const vec *>(y + s * a.y_row);
            const double w = a.weights[t * a.weights_stride + s];
#pragma unroll
            for (int e = 0; e < N; ++e) sum[e] = fma(w, (double)v[e], sum[e]);
        }
        vec out;
#pragma unroll
        for (int e = 0; e < N; ++e) out[e] = (float)sum[e];
        *reinterpret_cast<vec *>(a.dst + t * a.dst_stride + u) = out;
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
    if (!dst || dst_stride < nrows || dst_stride > lim || (add && (add_stride < nrows || add_stride > lim)))
        return (int)hipErrorInvalidValue;
    if (n_ids > 0 && (!y || !weights || y_token_stride < 0 || y_row_stride < 0 || y_token_stride > lim ||
                      y_row_stride > lim || weights_stride < n_ids || weights_stride > lim ||
                      (ids && (ids_stride < n_ids || ids_stride > lim))))
        return (int)hipErrorInvalidValue;
    if (add == dst && add_stride != dst_stride) return (int)hipErrorInvalidValue;
    const CombineArgs a = {y, weights, add, ids, dst, y_token_stride, y_row_stride, weights_stride, ids_stride,
                           add_stride, dst_stride, n_tokens, nrows, (int)n_ids};
    const bool wide = !(nrows % 4 || dst_stride % 4 || (uintptr_t)dst % 16 ||
                        (n_ids && (y_token_stride % 4 || y_row_stride % 4 || (uintptr_t)y % 16)) ||
                        (add && (add_stride % 4 || (uintptr_t)add % 16)));
    const int64_t units = n_tokens * (nrows / (wide ? 4 : 1));
    const dim3 grid((unsigned)std::min((units + THREADS - 1) / THREADS, (int64_t)1 << 20));
    if (wide)
        hipLaunchKernelGGL(combine_kernel<4>, grid, dim3(THREADS), 0, (hipStream_t)stream, a);
    else
        hipLaunchKernelGGL(combine_kernel<1>, grid, dim3(THREADS), 0, (hipStream_t)stream, a);
    return (int)hipGetLastError();
}
