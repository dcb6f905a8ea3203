// i8_quantize.hip -- what the 8-bit products need before them: rows of f32 as
// 8-bit integers with a scale each, and the pairs of (token, slot) grouped by
// experts.  Launches of latency: 24 rows of 4096 take 3.4 to 4 us; 4096 rows of 2048
// 11.5, and with the counts of 32768 pairs, in one, 12.9 (3.2 TB/s read and written),
// the pairs' places after them 8.0.  Many long rows are HBM bound: 4096 of 14336 take
// 59.9 us (4.9 TB/s).
#include <math.h>

#include <algorithm>

#include "i8.h"

using namespace i8;

namespace {

struct Rows {
    const float *x;
    int K;
    int64_t n_rows, x_stride;
    int8_t *q;
    int64_t q_stride;
    float *scale;
};

// TEAM threads a row, its values in registers between the maximum and the rounding: one read of memory, for rows of up to
// TEAM * V float4.  HBM bound on many rows, latency on few.  Workgroup `block` of `blocks` of BLOCK threads; `most` is for
// 2 * BLOCK / 64 values in LDS.
template <int BLOCK, int TEAM, int V>
__device__ __forceinline__ void quantize_rows(const Rows &a, int block, int blocks, uint32_t *most) {
    constexpr int TEAMS = BLOCK / TEAM, WAVES = BLOCK / 64;
    typedef uint32_t word __attribute__((aligned(1)));  // a store of 4 bytes need not be aligned
    const int team = threadIdx.x / TEAM, tid = threadIdx.x % TEAM, units = a.K / 4;
    int turn = 0;
    for (int64_t base = (int64_t)block * TEAMS; base < a.n_rows; base += (int64_t)blocks * TEAMS, turn ^= 1) {
        const int64_t r = base + team;
        const bool real = r < a.n_rows;
        const float *x = a.x + r * a.x_stride;
        int8_t *q = a.q + r * a.q_stride;
        uint32_t m = 0;
        float4 v[V];
        auto larger = [&](float4 u) {
            m = max(m, max(max(magnitude(u.x), magnitude(u.y)), max(magnitude(u.z), magnitude(u.w))));
        };
        const int end = real ? units : 0;
#pragma unroll
        for (int i = 0; i < V; ++i) {
            v[i] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            if (i * TEAM + tid < end) v[i] = four_at(x + 4 * (i * TEAM + tid));
        }
        // The up to three values behind the last four, a thread each.
        const int rest = 4 * units + tid;
        const float last = real && rest < a.K && tid < 3 ? x[rest] : 0.0f;
#pragma unroll
        for (int i = 0; i < V; ++i) larger(v[i]);
        m = max(m, magnitude(last));
        for (int k = V * TEAM + tid; k < end; k += TEAM) larger(four_at(x + 4 * k));  // rows longer than the registers: read twice
#pragma unroll
        for (int d = 32; d; d >>= 1) m = max(m, (uint32_t)__shfl_xor((int)m, d));
        if constexpr (TEAM > 64) {
            if ((threadIdx.x & 63) == 0) most[turn * WAVES + (threadIdx.x >> 6)] = m;
            __syncthreads();
#pragma unroll
            for (int w = 0; w < TEAM / 64; ++w) m = max(m, most[turn * WAVES + team * (TEAM / 64) + w]);
        }
        const Scale s(m);
#pragma unroll
        for (int i = 0; i < V; ++i)
            if (i * TEAM + tid < end) reinterpret_cast<word *>(q)[i * TEAM + tid] = s.four(v[i]);
        for (int k = V * TEAM + tid; k < end; k += TEAM) reinterpret_cast<word *>(q)[k] = s.four(four_at(x + 4 * k));
        if (real && rest < a.K && tid < 3) q[rest] = (int8_t)s.divided(last);
        if (real && tid == 0) a.scale[r] = s.value;
    }
}

template <int TEAM, int V>
__global__ __launch_bounds__(TEAM) void quantize_kernel(Rows a) {
    __shared__ uint32_t most[2 * (TEAM / 64)];
    quantize_rows<TEAM, TEAM, V>(a, blockIdx.x, gridDim.x, most);
}

template <int TEAM, int V>
int launch(const Rows &a, hipStream_t s) {
    hipLaunchKernelGGL((quantize_kernel<TEAM, V>), dim3((unsigned)std::min(a.n_rows, (int64_t)1 << 20)), dim3(TEAM), 0, s, a);
    return (int)hipGetLastError();
}

constexpr int GROUP_THREADS = 1024, PER = PAIR_CHUNK / GROUP_THREADS;

// The pairs of (token, slot) by experts: where a pair's column stands among its expert's does not matter to any result,
// so it is the order in which LDS counters are met.  A workgroup counts the experts of a chunk of pairs and notes each
// pair's place in its chunk.  With more than one chunk `place_kernel` goes on from the counts; with one, it is done at once.
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
__device__ __forceinline__ void count_pairs(const Pairs &a, int chunk, int *count, int2 *sums) {
    int id[PER], at[PER];
    count[threadIdx.x] = 0;
    load(a, chunk, id);
    __syncthreads();
#pragma unroll
    for (int i = 0; i < PER; ++i) at[i] = id[i] >= 0 ? atomicAdd(&count[id[i]], 1) : 0;
    __syncthreads();
    if constexpr (ONE) {
        const int total = count[threadIdx.x];
        __syncthreads();
        place(a, id, at, 0, 0, total, true, count, sums);
    } else {
        if ((int)threadIdx.x < a.n_as) a.counts[(int64_t)chunk * a.n_as + threadIdx.x] = count[threadIdx.x];
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const int p = chunk * PAIR_CHUNK + i * GROUP_THREADS + threadIdx.x;
            if (p < a.n_pairs) a.places[p] = (uint16_t)at[i];
        }
    }
}

// The first workgroups count pairs, the others quantize tokens meanwhile.
template <int TEAM, int V, bool ONE>
__global__ __launch_bounds__(GROUP_THREADS, 8) void prepare_kernel(Pairs a, int chunks, Rows tokens) {
    __shared__ int count[GROUP_THREADS];
    __shared__ int2 sums[GROUP_THREADS / 64];
    if ((int)blockIdx.x < chunks)
        count_pairs<ONE>(a, blockIdx.x, count, sums);
    else
        quantize_rows<GROUP_THREADS, TEAM, V>(tokens, blockIdx.x - chunks, gridDim.x - chunks, (uint32_t *)count);
}

template <int TEAM, int V>
void launch_prepare(const Pairs &a, int chunks, const Rows &tokens, hipStream_t s) {
    const int64_t blocks = tokens.n_rows ? (tokens.n_rows * TEAM + GROUP_THREADS - 1) / GROUP_THREADS : 0;
    const dim3 grid((unsigned)(chunks + std::min(blocks, (int64_t)1 << 18))), block(GROUP_THREADS);
    if (chunks == 1)
        hipLaunchKernelGGL((prepare_kernel<TEAM, V, true>), grid, block, 0, s, a, chunks, tokens);
    else
        hipLaunchKernelGGL((prepare_kernel<TEAM, V, false>), grid, block, 0, s, a, chunks, tokens);
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
    if (e < a.n_as) {
        const int chunks = gridDim.x;
        for (int c0 = 0; c0 < chunks; c0 += 8) {  // eight loads under way together
            int n[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) n[i] = a.counts[(int64_t)min(c0 + i, chunks - 1) * a.n_as + e];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                before += c0 + i < chunk ? n[i] : 0;
                total += c0 + i < chunks ? n[i] : 0;
            }
        }
    }
    place(a, id, at, chunk, before, total, chunk == 0, base, sums);
}

}  // namespace

int i8::quantize(const float *x, int64_t K, int64_t n_rows, int64_t x_stride, int8_t *q, int64_t q_stride, float *scale,
                 hipStream_t s) {
    const Rows a = {x, (int)K, n_rows, x_stride, q, q_stride, scale};
    if (K <= 1024) return launch<64, 4>(a, s);
    if (K <= 8192) return launch<256, 8>(a, s);
    return launch<1024, 4>(a, s);
}

int i8::group(const int32_t *ids, int64_t ids_stride, int n_pairs, int n_ids, int n_as, int per_slot, int bn,
              const Groups &to, float *dst, int64_t dst_stride, int64_t nrows, const float *x, int64_t K, int64_t n_rows,
              int64_t x_stride, int8_t *q, int64_t q_stride, float *scale, hipStream_t s) {
    const Pairs a = {ids, ids_stride, n_pairs, n_ids, n_as, per_slot, bn, to.col_src, to.col_dst, to.tiles, to.n_tiles,
                     to.counts, to.places, dst, dst_stride, nrows};
    const Rows tokens = {x, (int)K, x ? n_rows : 0, x_stride, q, q_stride, scale};
    const int chunks = (n_pairs + PAIR_CHUNK - 1) / PAIR_CHUNK;
    // Registers for two workgroups a CU: four float4 a thread, or two with what longer rows need beside them.
    if (K <= 1024)
        launch_prepare<64, 4>(a, chunks, tokens, s);
    else if (K <= 4096)
        launch_prepare<256, 4>(a, chunks, tokens, s);
    else
        launch_prepare<1024, 2>(a, chunks, tokens, s);
    const int e = (int)hipGetLastError();
    if (e || chunks == 1) return e;
    hipLaunchKernelGGL(place_kernel, dim3((unsigned)chunks), dim3(GROUP_THREADS), 0, s, a);
    return (int)hipGetLastError();
}

extern "C" int hip_qmm_quantize_i8(const float *x, int64_t K, int64_t n_rows, int64_t x_stride, int8_t *q,
                                   int64_t q_stride, float *scale, void *stream) {
    if (K < 1 || K > MAX_K || n_rows < 0 || n_rows > (1 << 24)) return (int)hipErrorInvalidValue;
    if (n_rows == 0) return 0;
    if (!x || !q || !scale || ((uintptr_t)x | (uintptr_t)scale) % 4 || x_stride < K || q_stride < K ||
        x_stride > MAX_STRIDE || q_stride > MAX_STRIDE)
        return (int)hipErrorInvalidValue;
    return quantize(x, K, n_rows, x_stride, q, q_stride, scale, (hipStream_t)stream);
}
