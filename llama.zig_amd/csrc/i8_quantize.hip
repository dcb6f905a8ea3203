// i8_quantize.hip -- what the 8-bit products need before them: rows of f32 as
// 8-bit integers with a scale each, and the pairs of (token, slot) grouped by
// experts.
#include <math.h>

#include <algorithm>

#include "i8.h"

using namespace i8;

namespace {

// A workgroup a row, its values in registers between the maximum and the rounding: one read of memory.  HBM bound on
// many rows, latency on few.  V float4 a thread; WIDE: rows of whole aligned float4.
template <int THREADS, int V, bool WIDE>
__global__ __launch_bounds__(THREADS) void quantize_kernel(const float *__restrict__ x0, int K, int64_t n_rows,
                                                           int64_t x_stride, int8_t *__restrict__ q0, int64_t q_stride,
                                                           float *__restrict__ scale) {
    __shared__ uint32_t most[2][THREADS / 64];
    const int tid = threadIdx.x;
    int turn = 0;
    for (int64_t r = blockIdx.x; r < n_rows; r += gridDim.x, turn ^= 1) {
        const float *x = x0 + r * x_stride;
        int8_t *q = q0 + r * q_stride;
        uint32_t m = 0;
        float4 v[V];
        auto load = [&](int k) {  // values 4 k .. 4 k + 3
            if (WIDE) return reinterpret_cast<const float4 *>(x)[k];
            float4 u = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            u.x = x[4 * k];
            if (4 * k + 1 < K) u.y = x[4 * k + 1];
            if (4 * k + 2 < K) u.z = x[4 * k + 2];
            if (4 * k + 3 < K) u.w = x[4 * k + 3];
            return u;
        };
        auto store = [&](int k, uint32_t b) {
            if (WIDE) {
                reinterpret_cast<uint32_t *>(q)[k] = b;
                return;
            }
            for (int i = 0; i < min(4, K - 4 * k); ++i) q[4 * k + i] = (int8_t)(b >> (8 * i));
        };
        auto larger = [&](float4 u) {
            m = max(m, max(max(magnitude(u.x), magnitude(u.y)), max(magnitude(u.z), magnitude(u.w))));
        };
        const int units = (K + 3) / 4;
#pragma unroll
        for (int i = 0; i < V; ++i) {
            v[i] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            if (i * THREADS + tid < units) v[i] = load(i * THREADS + tid);
        }
#pragma unroll
        for (int i = 0; i < V; ++i) larger(v[i]);
        for (int k = V * THREADS + tid; k < units; k += THREADS) larger(load(k));  // rows longer than the registers: read twice
#pragma unroll
        for (int d = 32; d; d >>= 1) m = max(m, (uint32_t)__shfl_xor((int)m, d));
        if ((tid & 63) == 0) most[turn][tid >> 6] = m;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < THREADS / 64; ++w) m = max(m, most[turn][w]);
        const Scale s(m);
#pragma unroll
        for (int i = 0; i < V; ++i)
            if (i * THREADS + tid < units) store(i * THREADS + tid, s.four(v[i]));
        for (int k = V * THREADS + tid; k < units; k += THREADS) store(k, s.four(load(k)));
        if (tid == 0) scale[r] = s.value;
    }
}

template <int THREADS, int V>
int launch(bool wide, const float *x, int K, int64_t n_rows, int64_t x_stride, int8_t *q, int64_t q_stride, float *scale,
           hipStream_t s) {
    const dim3 grid((unsigned)std::min(n_rows, (int64_t)1 << 20)), block(THREADS);
    if (wide)
        hipLaunchKernelGGL((quantize_kernel<THREADS, V, true>), grid, block, 0, s, x, K, n_rows, x_stride, q, q_stride, scale);
    else
        hipLaunchKernelGGL((quantize_kernel<THREADS, V, false>), grid, block, 0, s, x, K, n_rows, x_stride, q, q_stride, scale);
    return (int)hipGetLastError();
}

constexpr int GROUP_THREADS = 1024, PER = PAIR_CHUNK / GROUP_THREADS;

// The pairs of (token, slot) by experts: where a pair's column stands among its expert's does not matter to any result,
// so it is the order in which LDS counters are met.  A workgroup counts the experts of a chunk of pairs and notes each
// pair's place in its chunk.  With more than one chunk `place_kernel` goes on from the counts; with one, it is done here.
struct Pairs {
    const int32_t *ids;
    int64_t ids_stride;
    int n_pairs, n_ids, n_as, per_slot, bn;
    int32_t *col_src, *col_dst, *tiles, *n_tiles;
    int32_t *counts;    // [chunks][n_as]
    uint16_t *places;   // [n_pairs]
    float *dst;
    int64_t dst_stride, nrows;
};

// The sum of the values of lower threads, and all.
__device__ __forceinline__ int2 scan(int2 v, int2 *sums, int2 &all) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int2 s = v;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const int x = __shfl_up(s.x, d), y = __shfl_up(s.y, d);
        if (lane >= d) s.x += x, s.y += y;
    }
    if (lane == 63) sums[wave] = s;
    __syncthreads();
    int2 before = make_int2(s.x - v.x, s.y - v.y);
    all = make_int2(0, 0);
    for (int w = 0; w < GROUP_THREADS / 64; ++w) {
        const int2 u = sums[w];
        if (w < wave) before.x += u.x, before.y += u.y;
        all.x += u.x, all.y += u.y;
    }
    return before;
}

__device__ __forceinline__ void place(const Pairs &a, const int (&id)[PER], const int (&at)[PER], int chunk, int before,
                                      int total, bool tables, int *base, int2 *sums) {
    // Thread e: expert e, with `before` pairs in chunks before this one and `total` in all.
    const int e = threadIdx.x;
    int2 all;
    const int2 first = scan(make_int2(total, (total + a.bn - 1) / a.bn), sums, all);
    base[e] = first.x + before;
    if (tables) {
        for (int i = 0; i * a.bn < total; ++i)
            reinterpret_cast<int4 *>(a.tiles)[first.y + i] =
                make_int4(e, first.x + i * a.bn, first.x + min(total, (i + 1) * a.bn), 0);
        if (e == 0) *a.n_tiles = all.y;
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        const int p = chunk * PAIR_CHUNK + i * GROUP_THREADS + e;
        if (p < a.n_pairs && id[i] >= 0) {
            const int c = base[id[i]] + at[i];
            a.col_src[c] = a.per_slot ? p : (uint32_t)p / (uint32_t)a.n_ids;
            a.col_dst[c] = p;
        }
        // Rows of ids that are no expert's are cleared by the wave.
        for (unsigned long long none = __ballot(p < a.n_pairs && id[i] < 0); none; none &= none - 1) {
            float *row = a.dst + (int64_t)(p - (e & 63) + __ffsll((long long)none) - 1) * a.dst_stride;
            for (int64_t m = e & 63; m < a.nrows; m += 64) row[m] = 0.0f;
        }
    }
}

__device__ __forceinline__ void load(const Pairs &a, int chunk, int (&id)[PER]) {
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        const int p = chunk * PAIR_CHUNK + i * GROUP_THREADS + (int)threadIdx.x;
        id[i] = -1;
        if (p < a.n_pairs) {
            const int t = (uint32_t)p / (uint32_t)a.n_ids;
            const int x = a.ids[(int64_t)t * a.ids_stride + (p - t * a.n_ids)];
            if ((uint32_t)x < (uint32_t)a.n_as) id[i] = x;
        }
    }
}

template <bool ONE>
__global__ __launch_bounds__(GROUP_THREADS) void count_kernel(Pairs a) {
    __shared__ int count[GROUP_THREADS];
    __shared__ int2 sums[GROUP_THREADS / 64];
    int id[PER], at[PER];
    count[threadIdx.x] = 0;
    load(a, blockIdx.x, id);
    __syncthreads();
#pragma unroll
    for (int i = 0; i < PER; ++i) at[i] = id[i] >= 0 ? atomicAdd(&count[id[i]], 1) : 0;
    __syncthreads();
    if constexpr (ONE) {
        const int total = count[threadIdx.x];
        __syncthreads();
        place(a, id, at, 0, 0, total, true, count, sums);
    } else {
        if ((int)threadIdx.x < a.n_as) a.counts[(int64_t)blockIdx.x * a.n_as + threadIdx.x] = count[threadIdx.x];
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const int p = blockIdx.x * PAIR_CHUNK + i * GROUP_THREADS + threadIdx.x;
            if (p < a.n_pairs) a.places[p] = (uint16_t)at[i];
        }
    }
}

__global__ __launch_bounds__(GROUP_THREADS) void place_kernel(Pairs a) {
    __shared__ int base[GROUP_THREADS];
    __shared__ int2 sums[GROUP_THREADS / 64];
    const int chunk = blockIdx.x, e = threadIdx.x;
    int id[PER], at[PER];
    load(a, chunk, id);
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        const int p = chunk * PAIR_CHUNK + i * GROUP_THREADS + e;
        at[i] = p < a.n_pairs ? a.places[p] : 0;
    }
    int before = 0, total = 0;
    if (e < a.n_as)
        for (int c = 0; c < (int)gridDim.x; ++c) {
            const int n = a.counts[(int64_t)c * a.n_as + e];
            before += c < chunk ? n : 0;
            total += n;
        }
    place(a, id, at, chunk, before, total, chunk == 0, base, sums);
}

}  // namespace

int i8::quantize(const float *x, int64_t K, int64_t n_rows, int64_t x_stride, int8_t *q, int64_t q_stride, float *scale,
                 hipStream_t s) {
    const bool wide = !(K % 4 || x_stride % 4 || q_stride % 4 || (uintptr_t)x % 16 || (uintptr_t)q % 4);
    if (K <= 1024) return launch<64, 4>(wide, x, (int)K, n_rows, x_stride, q, q_stride, scale, s);
    if (K <= 8192) return launch<256, 8>(wide, x, (int)K, n_rows, x_stride, q, q_stride, scale, s);
    return launch<1024, 4>(wide, x, (int)K, n_rows, x_stride, q, q_stride, scale, s);
}

int i8::group(const int32_t *ids, int64_t ids_stride, int n_pairs, int n_ids, int n_as, int per_slot, int bn,
              const Groups &to, float *dst, int64_t dst_stride, int64_t nrows, hipStream_t s) {
    const Pairs a = {ids, ids_stride, n_pairs, n_ids, n_as, per_slot, bn, to.col_src, to.col_dst, to.tiles, to.n_tiles,
                     to.counts, to.places, dst, dst_stride, nrows};
    const dim3 block(GROUP_THREADS);
    if (n_pairs <= PAIR_CHUNK) {
        hipLaunchKernelGGL(count_kernel<true>, dim3(1), block, 0, s, a);
        return (int)hipGetLastError();
    }
    const dim3 grid((unsigned)((n_pairs + PAIR_CHUNK - 1) / PAIR_CHUNK));
    hipLaunchKernelGGL(count_kernel<false>, grid, block, 0, s, a);
    if (int e = (int)hipGetLastError()) return e;
    hipLaunchKernelGGL(place_kernel, grid, block, 0, s, a);
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
