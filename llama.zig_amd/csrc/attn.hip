// attn.hip -- attention over the paged key-value cache.
#include <math.h>

#include "kv_cache.h"

using namespace kvc;

namespace {

struct AttnArgs {
    Cache c;
    const float *q;
    float *dst;
    int64_t q_token, q_head, dst_token, dst_head;
    const int32_t *q_starts, *table, *lens;
    int64_t table_stride;
    int n_seqs, n_heads, group, max_q, n_tokens;
    float scale;
    int window, sinks;
};

// The queries of sequence s: rows [*first, *first + count), the last at position n - 1.
__device__ __forceinline__ int queries_of(const AttnArgs &a, int s, int *first, int *n) {
    int lo = s, hi = s + 1;
    if (a.q_starts) {
        lo = max(a.q_starts[s], 0);
        hi = min(a.q_starts[s + 1], a.n_tokens);
    }
    *first = lo;
    const int64_t most = a.table_stride << a.c.page_shift;
    *n = (int)min((int64_t)max(a.lens[s], 0), most);
    return max(hi - lo, 0);
}

template <bool BF16>
__global__ __launch_bounds__(64) void simple_kernel(AttnArgs a) {
    __shared__ float qs[256], ps[64];
    const int head = blockIdx.y, s = blockIdx.z, lane = threadIdx.x;
    int first, n;
    const int m = queries_of(a, s, &first, &n);
    const int D = a.c.head_dim, page = 1 << a.c.page_shift;
    const int64_t hoff = (int64_t)(head / a.group) * a.c.head_stride;
    for (int i = blockIdx.x; i < m; i += gridDim.x) {
        const int p = n - m + i;
        const float *q = a.q + (int64_t)(first + i) * a.q_token + head * a.q_head;
        __syncthreads();
        for (int d = lane; d < D; d += 64) qs[d] = q[d] * a.scale;
        __syncthreads();
        float top = -INFINITY, sum = 0.f, acc[4] = {0.f, 0.f, 0.f, 0.f};
        for (int j0 = 0; j0 <= p; j0 += 64) {
            const int j = j0 + lane;
            bool seen = j <= p && (a.window == 0 || p - j < a.window || j < a.sinks);
            int64_t at = 0;
            if (seen) {
                const int e = a.table[s * a.table_stride + (j >> a.c.page_shift)];
                seen = e >= 0 && e < a.c.n_pages;
                at = e * a.c.page_stride + hoff + (int64_t)(j & (page - 1)) * a.c.token_stride;
            }
            float score = -INFINITY;
            if (seen) {
                score = 0.f;
                for (int d = 0; d < D; ++d) score += qs[d] * from16<BF16>(a.c.k[at + d]);
            }
            float mx = score;
            for (int o = 32; o; o >>= 1) mx = fmaxf(mx, __shfl_xor(mx, o));
            if (!__any(seen)) continue;
            const float now = fmaxf(top, mx), base = now == -INFINITY ? 0.f : now;
            const float shrink = expf(top - base), w = seen ? expf(score - base) : 0.f;
            float t = w;
            for (int o = 32; o; o >>= 1) t += __shfl_xor(t, o);
            sum = sum * shrink + t;
            top = now;
            for (int v = 0; v < 4; ++v) acc[v] *= shrink;
            for (int l = 0; l < 64; ++l) {
                if (!__shfl((int)seen, l)) continue;
                const float wl = __shfl(w, l);
                const int64_t al = __shfl(at, l);
                for (int v = 0; v < 4; ++v)
                    if (v * 64 + lane < D) acc[v] += wl * from16<BF16>(a.c.v[al + v * 64 + lane]);
            }
        }
        float *o = a.dst + (int64_t)(first + i) * a.dst_token + head * a.dst_head;
        for (int v = 0; v < 4; ++v)
            if (v * 64 + lane < D) o[v * 64 + lane] = sum == 0.f ? 0.f : acc[v] / sum;
    }
    (void)ps;
}

}  // namespace

extern "C" size_t hip_qmm_attn_paged_workspace_size(const hip_qmm_kv_cache *cache, int64_t n_heads, int64_t n_seqs,
                                                    int64_t n_tokens, int64_t max_q, int64_t max_kv, int64_t window,
                                                    int64_t sinks) {
    (void)cache, (void)n_heads, (void)n_seqs, (void)n_tokens, (void)max_q, (void)max_kv, (void)window, (void)sinks;
    return 0;
}

extern "C" int hip_qmm_attn_paged(const hip_qmm_kv_cache *cache, const float *q, int64_t n_heads,
                                  int64_t q_token_stride, int64_t q_head_stride, const int32_t *q_starts,
                                  int64_t n_seqs, int64_t n_tokens, int64_t max_q, const int32_t *page_table,
                                  int64_t table_stride, const int32_t *kv_lens, int64_t max_kv, float scale,
                                  int64_t window, int64_t sinks, float *dst, int64_t dst_token_stride,
                                  int64_t dst_head_stride, void *workspace, size_t workspace_size, void *stream) {
    AttnArgs a = {};
    const int64_t lim = (int64_t)1 << 40;
    if (!take(cache, &a.c)) return (int)hipErrorInvalidValue;
    const int64_t H = a.c.n_kv_heads, D = a.c.head_dim;
    if (n_heads < 1 || n_heads > 65535 || n_heads % H || n_seqs < 0 || n_seqs > 65535 || n_tokens < 0 ||
        n_tokens > ((int64_t)1 << 23) || max_q < 0 || max_q > n_tokens || max_kv < 0 || !isfinite(scale) ||
        window < 0 || sinks < 0 || window > (1 << 30) || sinks > (1 << 30) || table_stride < 0 || table_stride > INT32_MAX)
        return (int)hipErrorInvalidValue;
    if (!q_starts && (n_tokens != n_seqs || (n_tokens > 0 && max_q < 1))) return (int)hipErrorInvalidValue;
    if (n_seqs == 0 || n_tokens == 0 || max_q == 0) return 0;
    if (!q || !dst || !kv_lens || (table_stride > 0 && !page_table)) return (int)hipErrorInvalidValue;
    if (((uintptr_t)q | (uintptr_t)dst) & 15 || ((q_token_stride | q_head_stride | dst_token_stride | dst_head_stride) & 3) ||
        q_token_stride < 0 || q_head_stride < 0 || dst_token_stride < 0 || dst_head_stride < 0 || q_token_stride > lim ||
        q_head_stride > lim || dst_token_stride > lim || dst_head_stride > lim || (n_heads > 1 && dst_head_stride < D) ||
        (n_tokens > 1 && dst_token_stride < (n_heads - 1) * dst_head_stride + D))
        return (int)hipErrorInvalidValue;
    a.q = q;
    a.dst = dst;
    a.q_token = q_token_stride;
    a.q_head = q_head_stride;
    a.dst_token = dst_token_stride;
    a.dst_head = dst_head_stride;
    a.q_starts = q_starts;
    a.table = page_table;
    a.lens = kv_lens;
    a.table_stride = table_stride;
    a.n_seqs = (int)n_seqs;
    a.n_heads = (int)n_heads;
    a.group = (int)(n_heads / H);
    a.max_q = (int)max_q;
    a.n_tokens = (int)n_tokens;
    a.scale = scale;
    a.window = (int)window;
    a.sinks = (int)sinks;
    (void)max_kv, (void)workspace, (void)workspace_size;
    hipStream_t s = (hipStream_t)stream;
    const dim3 grid((unsigned)max_q, (unsigned)n_heads, (unsigned)n_seqs);
    if (cache->type == HIP_QMM_TYPE_BF16)
        hipLaunchKernelGGL(simple_kernel<true>, grid, dim3(64), 0, s, a);
    else
        hipLaunchKernelGGL(simple_kernel<false>, grid, dim3(64), 0, s, a);
    return (int)hipGetLastError();
}
