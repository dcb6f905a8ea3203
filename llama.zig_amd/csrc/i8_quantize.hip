// i8_quantize.hip -- rows of f32 to 8-bit integers with a scale each, and the
// pairs of (token, slot) grouped by experts.
#include <math.h>

#include <algorithm>

#include "i8.h"

using namespace i8;

namespace {

constexpr int THREADS = 256;

// The largest magnitude; a NaN counts as infinity.
__device__ __forceinline__ float magnitude(float x) { return x != x ? INFINITY : fabsf(x); }

__global__ __launch_bounds__(THREADS) void quantize_kernel(const float *__restrict__ x0, int K, int64_t n_rows,
                                                           int64_t x_stride, int8_t *__restrict__ q0, int64_t q_stride,
                                                           float *__restrict__ scale) {
    __shared__ float most[THREADS / 64];
    for (int64_t r = blockIdx.x; r < n_rows; r += gridDim.x) {
    const float *x = x0 + r * x_stride;
    int8_t *q = q0 + r * q_stride;
    float m = 0.0f;
    for (int k = threadIdx.x; k < K; k += THREADS) m = fmaxf(m, magnitude(x[k]));
#pragma unroll
    for (int d = 32; d; d >>= 1) m = fmaxf(m, __shfl_xor(m, d));
    if ((threadIdx.x & 63) == 0) most[threadIdx.x >> 6] = m;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < THREADS / 64; ++w) m = fmaxf(m, most[w]);
    const float d = m / 127.0f;
    const bool usable = d > 0.0f && m < INFINITY;
    for (int k = threadIdx.x; k < K; k += THREADS)
        q[k] = usable ? (int8_t)fminf(fmaxf(rintf(x[k] / d), -127.0f), 127.0f) : (int8_t)0;
    if (threadIdx.x == 0) scale[r] = m < INFINITY ? d : NAN;
    __syncthreads();
    }
}

constexpr int GROUP_THREADS = 1024;

// Workgroup e finds the pairs of expert e in their order: it counts those of
// every expert (LDS atomics), and so knows where its columns and tiles start.
// Workgroup n_as clears the rows of ids that are no expert's.
__global__ __launch_bounds__(GROUP_THREADS) void group_kernel(const int32_t *__restrict__ ids, int64_t ids_stride,
                                                              int n_pairs, int n_ids, int n_as, int per_slot, int bn,
                                                              int32_t *__restrict__ col_src,
                                                              int32_t *__restrict__ col_dst, int32_t *__restrict__ tiles,
                                                              int32_t *__restrict__ n_tiles, float *__restrict__ dst,
                                                              int64_t dst_stride, int64_t nrows) {
    __shared__ int count[MAX_EXPERTS];
    __shared__ int before[GROUP_THREADS / 64], sums[2];
    const int tid = threadIdx.x, e = blockIdx.x, lane = tid & 63, wave = tid >> 6;
    auto id_of = [&](int p) {
        const int t = (uint32_t)p / (uint32_t)n_ids;
        return ids[(int64_t)t * ids_stride + (p - t * n_ids)];
    };
    if (e == n_as) {
        for (int p = wave; p < n_pairs; p += GROUP_THREADS / 64) {
            const int id = id_of(p);
            if ((uint32_t)id < (uint32_t)n_as) continue;
            float *row = dst + (int64_t)p * dst_stride;
            for (int64_t m = lane; m < nrows; m += 64) row[m] = 0.0f;
        }
        return;
    }
    if (tid < n_as) count[tid] = 0;
    if (tid < 2) sums[tid] = 0;
    __syncthreads();
    for (int p = tid; p < n_pairs; p += GROUP_THREADS) {
        const int id = id_of(p);
        if ((uint32_t)id < (uint32_t)n_as) atomicAdd(&count[id], 1);
    }
    __syncthreads();
    if (tid < n_as) {
        const int c = count[tid];
        if (tid < e && c) {
            atomicAdd(&sums[0], c);
            atomicAdd(&sums[1], (c + bn - 1) / bn);
        }
    }
    __syncthreads();
    const int first = sums[0], tile = sums[1], mine = count[e];
    if (e == n_as - 1 && tid == 0) *n_tiles = tile + (mine + bn - 1) / bn;
    for (int i = tid; i * bn < mine; i += GROUP_THREADS) {
        int32_t *t = tiles + 4 * (int64_t)(tile + i);
        t[0] = e, t[1] = first + i * bn, t[2] = first + min(mine, (i + 1) * bn), t[3] = 0;
    }
    int at = first;
    for (int base = 0; base < n_pairs; base += GROUP_THREADS) {
        const int p = base + tid;
        const bool is = p < n_pairs && id_of(p) == e;
        const unsigned long long who = __ballot(is);
        __syncthreads();  // the last round's reads of `before`
        if (lane == 0) before[wave] = __popcll(who);
        __syncthreads();
        int c = at;
        for (int w = 0; w < GROUP_THREADS / 64; ++w) {
            if (w < wave) c += before[w];
            at += before[w];
        }
        if (is) {
            c += __popcll(who & ((1ull << lane) - 1));
            const int t = (uint32_t)p / (uint32_t)n_ids;
            col_src[c] = per_slot ? p : t;
            col_dst[c] = p;
        }
    }
}

}  // namespace

int i8::quantize(const float *x, int64_t K, int64_t n_rows, int64_t x_stride, int8_t *q, int64_t q_stride, float *scale,
                 hipStream_t s) {
    hipLaunchKernelGGL(quantize_kernel, dim3((unsigned)std::min(n_rows, (int64_t)1 << 20)), dim3(THREADS), 0, s, x, (int)K, n_rows,
                       x_stride, q, q_stride,
                       scale);
    return (int)hipGetLastError();
}

int i8::group(const int32_t *ids, int64_t ids_stride, int64_t n_tokens, int64_t n_ids, int64_t n_as, int64_t ne11,
              int bn, int32_t *col_src, int32_t *col_dst, int32_t *tiles, int32_t *n_tiles, float *dst,
              int64_t dst_stride, int64_t nrows, hipStream_t s) {
    hipLaunchKernelGGL(group_kernel, dim3((unsigned)n_as + 1), dim3(GROUP_THREADS), 0, s, ids, ids_stride,
                       (int)(n_tokens * n_ids), (int)n_ids, (int)n_as, (int)(ne11 > 1), bn, col_src, col_dst, tiles,
                       n_tiles, dst, dst_stride, nrows);
    return (int)hipGetLastError();
}

extern "C" int hip_qmm_quantize_i8(const float *x, int64_t K, int64_t n_rows, int64_t x_stride, int8_t *q,
                                   int64_t q_stride, float *scale, void *stream) {
    if (K < 1 || K > MAX_K || n_rows < 0 || n_rows > (1 << 24)) return (int)hipErrorInvalidValue;
    if (n_rows == 0) return 0;
    if (!x || !q || !scale || x_stride < K || q_stride < K || x_stride > MAX_STRIDE || q_stride > MAX_STRIDE)
        return (int)hipErrorInvalidValue;
    return quantize(x, K, n_rows, x_stride, q, q_stride, scale, (hipStream_t)stream);
}
