// kv_pages.hip -- upkeep of the paged key-value cache: page copies, and the
// move of all pages in use to the front of the pool with the rewrite of the
// page tables.
//
// Both are HBM streams of 16-byte units.  The compaction's plan (which pages
// are in use, how many, what goes where) is one workgroup's work on a bitmap
// in LDS, and its moves a second launch whose work list the first wrote: the
// host never waits.
#include "kv_cache.h"

using namespace kvc;

namespace {

constexpr int COPY_THREADS = 256;
constexpr int PLAN_THREADS = 1024;
constexpr int64_t MAX_PLAN_PAGES = 1 << 20;

// The first `tokens` tokens of one head of a page: K and V alike.
__device__ __forceinline__ void copy_head(const Cache &c, uint16_t *base, int64_t from, int64_t to, int tokens) {
    const int units = c.head_dim >> 3;
    const uint16_t *s = base + from;
    uint16_t *d = base + to;
    for (int i = threadIdx.x; i < tokens * units; i += COPY_THREADS) {
        const int t = i / units, u = i - t * units;
        const int64_t at = t * c.token_stride + u * 8;
        *reinterpret_cast<uint4 *>(d + at) = *reinterpret_cast<const uint4 *>(s + at);
    }
}

// Workgroup (head, keys or values, pair).
__global__ __launch_bounds__(COPY_THREADS) void copy_kernel(Cache c, const int32_t *__restrict__ src,
                                                            const int32_t *__restrict__ dst,
                                                            const int32_t *__restrict__ n_tokens, int64_t n_copies) {
    for (int64_t i = blockIdx.x; i < n_copies; i += gridDim.x) {
        const int from = src[i], to = dst[i];
        if (from < 0 || to < 0 || from >= c.n_pages || to >= c.n_pages) continue;
        const int page = 1 << c.page_shift;
        const int tokens = n_tokens ? min(n_tokens[i], page) : page;
        for (int h = blockIdx.y; h < c.n_kv_heads; h += gridDim.y) {
            const int64_t head = (int64_t)h * c.head_stride;
            copy_head(c, blockIdx.z ? c.v : c.k, from * c.page_stride + head, to * c.page_stride + head, tokens);
        }
    }
}

// The workspace of a compaction: a header, the k-th unused page below n_live
// (hole) with the k-th page in use from n_live on (from), and per page its k.
struct Plan {
    int32_t *n_live, *n_moves, *hole, *from, *rank;
};

__host__ __device__ inline Plan plan_at(void *ws, int64_t n_pages) {
    int32_t *p = (int32_t *)ws;
    return {p, p + 1, p + 64, p + 64 + n_pages, p + 64 + 2 * n_pages};
}

// Entry (row, column) of the tables: its page if it is in use, else -1.
__device__ __forceinline__ int entry_of(const int32_t *table, int64_t stride, const int32_t *lens, int64_t row,
                                        int64_t col, int page_shift, int n_pages) {
    const int64_t n = lens[row];
    if ((col << page_shift) >= n) return -1;
    const int e = table[row * stride + col];
    return e >= 0 && e < n_pages ? e : -1;
}

// Sum over the workgroup of one value per thread, and the sum over the
// threads before this one.
__device__ __forceinline__ int block_scan(int v, int *part, int *total) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int s = v;
    for (int o = 1; o < 64; o <<= 1) {
        const int u = __shfl_up(s, o);
        if (lane >= o) s += u;
    }
    __syncthreads();
    if (lane == 63) part[wave] = s;
    __syncthreads();
    int before = 0, all = 0;
    for (int w = 0; w < PLAN_THREADS / 64; ++w) {
        if (w < wave) before += part[w];
        all += part[w];
    }
    *total = all;
    return before + s - v;
}

// One workgroup.  Thread t owns the bitmap's words [t*per, (t+1)*per).
__global__ __launch_bounds__(PLAN_THREADS) void plan_kernel(const int32_t *__restrict__ table, int64_t stride,
                                                            int64_t width, const int32_t *__restrict__ lens,
                                                            int64_t n_seqs, int page_shift, int n_pages, void *ws,
                                                            int32_t *n_live_out) {
    extern __shared__ uint32_t used[];
    __shared__ int part[PLAN_THREADS / 64];
    const int words = (n_pages + 31) / 32, per = (words + PLAN_THREADS - 1) / PLAN_THREADS;
    const Plan p = plan_at(ws, n_pages);
    for (int w = threadIdx.x; w < words; w += PLAN_THREADS) used[w] = 0;
    __syncthreads();
    // A wave takes ROWS rows at a time, whose loads are in flight together.
    constexpr int ROWS = 4, WAVES = PLAN_THREADS / 64;
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    for (int64_t row = wave * ROWS; row < n_seqs; row += WAVES * ROWS) {
        int64_t n[ROWS], most = 0;
#pragma unroll
        for (int i = 0; i < ROWS; ++i) {
            const int64_t len = row + i < n_seqs ? lens[row + i] : 0;
            n[i] = len <= 0 ? 0 : ((len - 1) >> page_shift) + 1;
            if (n[i] > width) n[i] = width;
            most = most > n[i] ? most : n[i];
        }
        for (int64_t col = lane; col < most; col += 64) {
            int e[ROWS];
#pragma unroll
            for (int i = 0; i < ROWS; ++i) e[i] = col < n[i] ? table[(row + i) * stride + col] : -1;
#pragma unroll
            for (int i = 0; i < ROWS; ++i)
                if (e[i] >= 0 && e[i] < n_pages) atomicOr(&used[e[i] >> 5], 1u << (e[i] & 31));
        }
    }
    __syncthreads();
    const int w0 = min(words, (int)threadIdx.x * per), w1 = min(words, w0 + per);
    int mine = 0, live, moves;
    for (int w = w0; w < w1; ++w) mine += __popc(used[w]);
    const int before = block_scan(mine, part, &live);
    // Of pages below n_live, those unused; from it on, those in use: as many.
    // Thread t's count of unused pages below n_live before its words: pages
    // there, less those in use; pages in use from n_live on likewise, by its own scan.
    int high = 0;
    for (int w = w0; w < w1; ++w)
        for (uint32_t b = used[w]; b; b &= b - 1) high += w * 32 + __ffs(b) - 1 >= live;
    const int high_before = block_scan(high, part, &moves);
    int hole = min(w0 * 32, live) - (before - high_before), k = high_before;
    for (int w = w0; w < w1; ++w) {
        const uint32_t bits = used[w];
        for (int b = 0; b < 32; ++b) {
            const int page = w * 32 + b;
            if (page >= n_pages) break;
            const bool in_use = bits >> b & 1;
            if (page < live && !in_use) p.hole[hole++] = page;
            if (page >= live && in_use) {
                p.rank[page] = k;
                p.from[k++] = page;
            }
        }
    }
    if (threadIdx.x == 0) {
        *p.n_live = live;
        *p.n_moves = moves;
        *n_live_out = live;
    }
}

// The first table_blocks workgroups rewrite the tables, the others move pages.
__global__ __launch_bounds__(COPY_THREADS) void apply_kernel(Cache c, const int32_t *table, int64_t stride,
                                                             int64_t width, const int32_t *__restrict__ lens,
                                                             int64_t n_seqs, int32_t *out, int64_t out_stride,
                                                             void *ws, int table_blocks) {
    const Plan p = plan_at(ws, c.n_pages);
    const int live = *p.n_live;
    if ((int)blockIdx.x < table_blocks) {
        for (int64_t i = (int64_t)blockIdx.x * COPY_THREADS + threadIdx.x; i < n_seqs * width;
             i += (int64_t)table_blocks * COPY_THREADS) {
            const int64_t row = i / width, col = i - row * width;
            const int e = entry_of(table, stride, lens, row, col, c.page_shift, c.n_pages);
            out[row * out_stride + col] = e >= live ? p.hole[p.rank[e]] : e;
        }
        return;
    }
    const int64_t work = (int64_t)*p.n_moves * c.n_kv_heads * 2;
    for (int64_t i = blockIdx.x - table_blocks; i < work; i += gridDim.x - table_blocks) {
        const int64_t m = i / (c.n_kv_heads * 2);
        const int r = (int)(i - m * c.n_kv_heads * 2);
        const int64_t head = (int64_t)(r >> 1) * c.head_stride;
        copy_head(c, r & 1 ? c.v : c.k, p.from[m] * c.page_stride + head, p.hole[m] * c.page_stride + head,
                  1 << c.page_shift);
    }
}

}  // namespace

extern "C" int hip_qmm_kv_copy_pages(const hip_qmm_kv_cache *cache, const int32_t *src, const int32_t *dst,
                                     const int32_t *n_tokens, int64_t n_copies, void *stream) {
    Cache c;
    if (!take(cache, &c) || n_copies < 0 || (n_copies > 0 && (!src || !dst))) return (int)hipErrorInvalidValue;
    if (n_copies == 0) return 0;
    const dim3 grid((unsigned)(n_copies < 65536 ? n_copies : 65536), (unsigned)c.n_kv_heads, 2);
    hipLaunchKernelGGL(copy_kernel, grid, dim3(COPY_THREADS), 0, (hipStream_t)stream, c, src, dst, n_tokens, n_copies);
    return (int)hipGetLastError();
}

extern "C" size_t hip_qmm_kv_compact_workspace_size(const hip_qmm_kv_cache *cache) {
    Cache c;
    if (!take(cache, &c) || c.n_pages > MAX_PLAN_PAGES) return 0;
    return (64 + 3 * (size_t)c.n_pages) * sizeof(int32_t);
}

extern "C" int hip_qmm_kv_compact(const hip_qmm_kv_cache *cache, const int32_t *page_table, int64_t table_stride,
                                  int64_t table_width, const int32_t *kv_lens, int64_t n_seqs, int32_t *table_out,
                                  int64_t out_stride, int32_t *n_live, void *workspace, size_t workspace_size,
                                  void *stream) {
    Cache c;
    if (!take(cache, &c) || c.n_pages > MAX_PLAN_PAGES || n_seqs < 0 || table_width < 0 ||
        table_stride < table_width || out_stride < table_width || !n_live || !workspace ||
        ((uintptr_t)workspace & 3) || workspace_size < hip_qmm_kv_compact_workspace_size(cache))
        return (int)hipErrorInvalidValue;
    if (n_seqs > 0 && table_width > 0 && (!page_table || !kv_lens || !table_out)) return (int)hipErrorInvalidValue;
    if (table_width > INT32_MAX || n_seqs > INT32_MAX || out_stride > ((int64_t)1 << 40) ||
        table_stride > ((int64_t)1 << 40) || (page_table == table_out && table_stride != out_stride))
        return (int)hipErrorInvalidValue;
    hipStream_t s = (hipStream_t)stream;
    const size_t lds = (size_t)(c.n_pages + 31) / 32 * 4;
    hipLaunchKernelGGL(plan_kernel, dim3(1), dim3(PLAN_THREADS), lds, s, page_table, table_stride, table_width, kv_lens,
                       n_seqs, c.page_shift, c.n_pages, workspace, n_live);
    const int e = (int)hipGetLastError();
    if (e) return e;
    const int64_t entries = n_seqs * table_width;
    const int table_blocks = (int)(entries / COPY_THREADS < 256 ? entries / COPY_THREADS + 1 : 256);
    const int64_t most = (entries < c.n_pages / 2 ? entries : c.n_pages / 2) * c.n_kv_heads * 2;  // moves x heads x {K, V}
    const int blocks = table_blocks + (int)(most < 8192 ? most : 8192) + 1;
    hipLaunchKernelGGL(apply_kernel, dim3((unsigned)blocks), dim3(COPY_THREADS), 0, s, c, page_table, table_stride,
                       table_width, kv_lens, n_seqs, table_out, out_stride, workspace, table_blocks);
    return (int)hipGetLastError();
}
