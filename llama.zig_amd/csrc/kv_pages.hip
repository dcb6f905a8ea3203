// kv_pages.hip -- upkeep of the paged key-value cache: page copies, and the
// move of all pages in use to the front of the pool with the rewrite of the
// page tables.
//
// Both are HBM streams of 16-byte units.  The compaction's plan (which pages
// are in use, how many, what goes where) is one workgroup's work on a bitmap in
// LDS.  For small pools every workgroup makes it for itself before its share of
// the moves; for large ones the moves are a second launch whose work list the
// first wrote.  The host never waits.
#include <algorithm>

#include "kv_cache.h"

using namespace kvc;

namespace {

typedef uint32_t v4u __attribute__((ext_vector_type(4)));

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

// A pool's page whose heads and tokens leave no gaps is one run of 16-byte
// units: a workgroup copies PART of them, four per thread in flight (compaction
// of 4096 pages, 134 MB: 34 us; head by head, one in flight, 42).
constexpr int PART = 4 * COPY_THREADS;

int run_units(const Cache &c) {
    const int64_t n = (int64_t)c.n_kv_heads << c.page_shift;
    const bool dense = (n - 1) * c.head_dim == (c.n_kv_heads - 1) * c.head_stride + ((1 << c.page_shift) - 1) * c.token_stride;
    return dense && n * c.head_dim / 8 < (1 << 30) ? (int)(n * c.head_dim / 8) : 0;
}

__device__ __forceinline__ void copy_run(const uint16_t *from, uint16_t *to, int units, int part) {
    const v4u *s = reinterpret_cast<const v4u *>(from);
    v4u *d = reinterpret_cast<v4u *>(to);
    int i = part * PART + threadIdx.x;
    if (i + 3 * COPY_THREADS < units) {
        v4u v[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) v[k] = s[i + k * COPY_THREADS];
#pragma unroll
        for (int k = 0; k < 4; ++k) d[i + k * COPY_THREADS] = v[k];
    } else {
        for (const int end = min(units, (part + 1) * PART); i < end; i += COPY_THREADS) d[i] = s[i];
    }
}

// The moves hole[m] <- from[m], m < moves, by all workgroups from `first` on; run: run_units.
template <class Index>
__device__ __forceinline__ void move_pages(const Cache &c, const Index *from, const Index *hole, int moves, int run,
                                           int first, int step) {
    const int pieces = run ? (run + PART - 1) / PART * 2 : c.n_kv_heads * 2;
    for (int64_t i = first; i < (int64_t)moves * pieces; i += step) {
        const int m = (int)(i / pieces), r = (int)(i - (int64_t)m * pieces);
        uint16_t *pool = r & 1 ? c.v : c.k;
        const int64_t s = from[m] * c.page_stride, d = hole[m] * c.page_stride;
        if (run) copy_run(pool + s, pool + d, run, r >> 1);
        else copy_head(c, pool, s + (r >> 1) * c.head_stride, d + (r >> 1) * c.head_stride, 1 << c.page_shift);
    }
}

// Workgroup (copy, head, keys or values): bound by the launch where only the
// last pages of some sequences are copied (64 of them, 4.5 MB: 2.6 us).
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
                                                             void *ws, int table_blocks, int run) {
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
    move_pages(c, p.from, p.hole, *p.n_moves, run, blockIdx.x - table_blocks, gridDim.x - table_blocks);
}

// Both for small pools in one launch: every workgroup makes the whole plan for
// itself, in LDS, and then rewrites its share of the tables and moves its share
// of the pages.  4096 pages, 1000 of them moving (134 MB): 34 us, 37 in two
// launches; the moves alone are 25 at the rate of a large copy, a plan 6.
constexpr int SMALL_PAGES = 8192, SMALL_ENTRIES = 16384;

__global__ __launch_bounds__(COPY_THREADS) void small_kernel(Cache c, const int32_t *__restrict__ table, int64_t stride,
                                                             int width, const int32_t *__restrict__ lens, int n_seqs,
                                                             int32_t *__restrict__ out, int64_t out_stride,
                                                             int32_t *n_live_out, int run) {
    constexpr int WORDS = SMALL_PAGES / 32, WAVES = COPY_THREADS / 64;
    static_assert(WORDS == COPY_THREADS, "a word per thread");
    __shared__ uint32_t used[WORDS];
    __shared__ uint16_t hole[SMALL_PAGES / 2], from[SMALL_PAGES / 2], high_before[WORDS];
    __shared__ int part[2][WAVES];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, entries = n_seqs * width;
    used[tid] = 0;
    __syncthreads();
#pragma unroll 8
    for (int i = tid; i < entries; i += COPY_THREADS) {
        const int row = i / width, col = i - row * width;
        const int n = lens[row], e = table[row * stride + col];  // both in flight
        if (((int64_t)col << c.page_shift) < n && e >= 0 && e < c.n_pages) atomicOr(&used[e >> 5], 1u << (e & 31));
    }
    __syncthreads();
    const uint32_t bits = used[tid];
    // Sums over the threads before this one, and over all, of two counts in turn.
    auto scan = [&](int v, int which, int *total) {
        int s = v;
        for (int o = 1; o < 64; o <<= 1) {
            const int u = __shfl_up(s, o);
            if (lane >= o) s += u;
        }
        if (lane == 63) part[which][wave] = s;
        __syncthreads();
        int before = s - v, all = 0;
        for (int w = 0; w < WAVES; ++w) {
            if (w < wave) before += part[which][w];
            all += part[which][w];
        }
        *total = all;
        return before;
    };
    int live, moves;
    const int before = scan(__popc(bits), 0, &live);
    const int page0 = tid * 32, below = min(max(live - page0, 0), 32);  // of this word's pages, those below n_live
    const uint32_t low = below == 32 ? ~0u : (1u << below) - 1;
    const int high = scan(__popc(bits & ~low), 1, &moves);
    high_before[tid] = (uint16_t)high;
    // The unused pages below n_live before this word, and the pages in use from n_live on.
    int h = min(page0, live) - (before - high), k = high;
    for (uint32_t b = ~bits & low; b; b &= b - 1) hole[h++] = (uint16_t)(page0 + __ffs(b) - 1);
    for (uint32_t b = bits & ~low; b; b &= b - 1) from[k++] = (uint16_t)(page0 + __ffs(b) - 1);
    __syncthreads();
    if (blockIdx.x == 0 && tid == 0) *n_live_out = live;
    for (int i = blockIdx.x * COPY_THREADS + tid; i < entries; i += gridDim.x * COPY_THREADS) {
        const int row = i / width, col = i - row * width;
        int e = entry_of(table, stride, lens, row, col, c.page_shift, c.n_pages);
        if (e >= live) {
            const int w = e >> 5, first = max(live - w * 32, 0);  // live <= e: first < 32
            e = hole[high_before[w] + __popc(used[w] & ((1u << (e & 31)) - 1) & (~0u << first))];
        }
        out[row * out_stride + col] = e;
    }
    move_pages(c, from, hole, moves, run, blockIdx.x, gridDim.x);
}

// Whole pages that are runs: workgroup (part of a page, copy, keys or values).
__global__ __launch_bounds__(COPY_THREADS) void copy_run_kernel(Cache c, const int32_t *__restrict__ src,
                                                                const int32_t *__restrict__ dst, int64_t n_copies,
                                                                int run) {
    for (int64_t i = blockIdx.y; i < n_copies; i += gridDim.y) {
        const int from = src[i], to = dst[i];
        if (from < 0 || to < 0 || from >= c.n_pages || to >= c.n_pages) continue;
        uint16_t *pool = blockIdx.z ? c.v : c.k;
        copy_run(pool + from * c.page_stride, pool + to * c.page_stride, run, blockIdx.x);
    }
}

}  // namespace

extern "C" int hip_qmm_kv_copy_pages(const hip_qmm_kv_cache *cache, const int32_t *src, const int32_t *dst,
                                     const int32_t *n_tokens, int64_t n_copies, void *stream) {
    Cache c;
    if (!take(cache, &c) || n_copies < 0 || (n_copies > 0 && (!src || !dst))) return (int)hipErrorInvalidValue;
    if (n_copies == 0) return 0;
    const int run = run_units(c);
    if (!n_tokens && run) {
        const dim3 grid((unsigned)((run + PART - 1) / PART), (unsigned)std::min(n_copies, (int64_t)65535), 2);
        hipLaunchKernelGGL(copy_run_kernel, grid, dim3(COPY_THREADS), 0, (hipStream_t)stream, c, src, dst, n_copies, run);
        return (int)hipGetLastError();
    }
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
    if (table_width == 0) n_seqs = 0;  // nothing in use; the lengths, which may be absent then, are not read
    hipStream_t s = (hipStream_t)stream;
    // In one launch, unless a workgroup would read rows of the table that another has rewritten, or every one a
    // large table.
    const uintptr_t in0 = (uintptr_t)page_table, out0 = (uintptr_t)table_out;
    const uintptr_t in1 = in0 + (size_t)n_seqs * (size_t)table_stride * 4;
    const uintptr_t out1 = out0 + (size_t)n_seqs * (size_t)out_stride * 4;
    if (c.n_pages <= SMALL_PAGES && n_seqs <= SMALL_ENTRIES && table_width <= SMALL_ENTRIES &&
        n_seqs * table_width <= SMALL_ENTRIES && (in1 <= out0 || out1 <= in0)) {
        const int64_t units = c.n_pages / 2 * c.n_kv_heads * 2 + 1;
        hipLaunchKernelGGL(small_kernel, dim3((unsigned)std::min(units, (int64_t)1024)), dim3(COPY_THREADS), 0, s, c,
                           page_table, table_stride, (int)table_width, kv_lens, (int)n_seqs, table_out, out_stride, n_live,
                           run_units(c));
        return (int)hipGetLastError();
    }
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
                       table_width, kv_lens, n_seqs, table_out, out_stride, workspace, table_blocks, run_units(c));
    return (int)hipGetLastError();
}
