/*
 * ggml_hip_attn.h -- C ABI of the operators between a decoder layer's
 * quantized projections, in libggml_hip_qmm.so: rotary positions with the
 * store into a paged key-value cache, attention over that cache, and the
 * upkeep of its pages.
 *
 * Conventions are those of ggml_hip_qmm.h: device pointers unless a comment
 * says host, activations f32, asynchronous on `stream`, no allocation, scratch
 * from the caller, 0 or a hipError_t back (hipErrorInvalidValue = 1 for what an
 * entry does not take, before anything is launched).
 */
#ifndef GGML_HIP_ATTN_H
#define GGML_HIP_ATTN_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* ggml type ids of the cache's elements. */
#define HIP_QMM_TYPE_F16 1
#define HIP_QMM_TYPE_BF16 30

/*
 * One layer's key-value cache (a host structure).  k and v are pools of
 * n_pages pages; the element of dimension d of token t (0 <= t < page_size)
 * of page p for key-value head h is at
 * p*page_stride + h*head_stride + t*token_stride + d, in elements, the same in
 * both.  head_dim is a multiple of 8 up to 256, page_size a power of two from
 * 16 to 65536; k, v 16-byte aligned and the strides multiples of 8 elements;
 * pages, and the heads and tokens of a page, do not overlap; token_stride is
 * at most 2^27.  At most 2^31 - 1 tokens in all.
 */
typedef struct hip_qmm_kv_cache {
    void *k, *v;
    int32_t type; /* HIP_QMM_TYPE_F16 or _BF16 */
    int32_t n_kv_heads, page_size, head_dim;
    int64_t n_pages;
    int64_t page_stride, head_stride, token_stride;
} hip_qmm_kv_cache;

/* Which two elements of a head a rotation takes: x[2i], x[2i+1], or
 * x[i], x[i + n_dims/2] (ggml's rope modes of these values). */
#define HIP_QMM_ROPE_INTERLEAVED 0
#define HIP_QMM_ROPE_HALF 2

/*
 * The rotations of a model, computed on the host once: steps[i], i <
 * n_dims/2, is the turn that one position adds to pair i, in units of 2^-64
 * turns modulo one turn, so that the turn of any position is exact up to that
 * rounding (an f32 angle is off by position * 2^-24).  Pair i turns by
 *   f = freq_base^(-2i/n_dims) / freq_factors[i] (host; NULL: 1)
 * radians a position without scaling, by f*freq_scale when interpolated, and
 * by a mix of the two with ext_factor > 0 (YaRN): the share of f falls from
 * ext_factor to 0 between the pairs that turn beta_fast and beta_slow times
 * over n_ctx_orig positions.  *mscale is attn_factor, times 1 + 0.1
 * ln(1/freq_scale) with ext_factor > 0.  steps and mscale are host memory;
 * the kernels take steps from device memory.  n_dims even, 2..256.
 */
int hip_qmm_rope_steps(int n_dims, double freq_base, double freq_scale, double ext_factor, double attn_factor,
                       double beta_fast, double beta_slow, int64_t n_ctx_orig, const float *freq_factors,
                       int64_t *steps, float *mscale);

/*
 * dst[t][h] = x[t][h] with its first n_dims elements rotated by position
 * pos[t]: each pair (a, b) becomes mscale * (a cos - b sin, a sin + b cos); the
 * other head_dim - n_dims elements are copied.  Token t's head h starts at
 * x + t*x_token_stride + h*x_head_stride (floats; elements contiguous), dst
 * likewise.  dst may be x with the same strides; other overlap is not allowed.
 * Positions may be negative.  head_dim at most 1024, n_dims even and at most
 * 256 and head_dim, n_tokens at most 2^23.
 */
int hip_qmm_rope_f32(const float *x, int64_t n_tokens, int64_t n_heads, int64_t head_dim, int64_t x_token_stride,
                     int64_t x_head_stride, const int32_t *pos, const int64_t *steps, int n_dims, int layout,
                     float mscale, float *dst, int64_t dst_token_stride, int64_t dst_head_stride, void *stream);

/*
 * What a step does between the q/k/v projections and attention, in one
 * launch: hip_qmm_rope_f32 of q (n_heads heads) into q_dst, and the same
 * rotation of k and the plain v (the cache's n_kv_heads heads; shared strides)
 * rounded to the cache's type at slot slots[t] = page*page_size + token.  A slot
 * outside the cache stores nothing; two tokens with one slot store one of the
 * two in each place.  q may be NULL (n_heads = 0) to store only.
 */
int hip_qmm_rope_kv_store(const float *q, int64_t n_heads, int64_t q_token_stride, int64_t q_head_stride,
                          const float *k, const float *v, int64_t kv_token_stride, int64_t kv_head_stride,
                          int64_t n_tokens, const int32_t *pos, const int64_t *steps, int n_dims, int layout,
                          float mscale, float *q_dst, int64_t dst_token_stride, int64_t dst_head_stride,
                          const hip_qmm_kv_cache *cache, const int32_t *slots, void *stream);

/*
 * Attention of the newest tokens of n_seqs sequences over the paged cache.
 * Sequence s holds n = kv_lens[s] tokens, token j in page
 * page_table[s*table_stride + j / page_size] (n_seqs rows of table_stride
 * entries; lengths are cut to table_stride*page_size and to 2^30; negative ones
 * count as 0), and its last m have queries: rows q_starts[s] <= t <
 * q_starts[s+1] of q, or row s alone (m = 1) with q_starts NULL.  The keys and
 * values of the new tokens are in the cache already.  The query of position p
 * sees token j if
 *   j <= p  and  (window == 0  or  p - j < window  or  j < sinks)
 * and j's page lies in [0, n_pages): pages that fell out of the window may be
 * freed and their entries set to -1.  With head h's keys and values in
 * key-value head h / (n_heads / n_kv_heads):
 *   dst[t][h] = sum_j w_j v_j / sum_j w_j,   w_j = exp(scale * q[t][h].k_j)
 * over the tokens it sees, a zero row where it sees none (as for a query at a
 * negative position, where m > n) or only scores of -infinity.  What hidden
 * tokens hold, NaN and infinities too, does not matter; what is seen counts as
 * IEEE arithmetic has it (an infinite key gives a weight of 0 or a row of NaN),
 * and a query that is not finite gives a row of NaN.  Results are f32 throughout: q and w enter the matrix
 * cores as sums of f16 or bf16 parts that hold 22 bits and more.
 * q_starts ascends from 0 or more to n_tokens or less; max_q is at least the
 * largest m and at most n_tokens; max_kv, the largest length in the host's
 * knowledge, only plans the work.  n_heads a multiple of n_kv_heads; q and dst
 * 16-byte aligned with strides that are multiples of 4 floats, dst's tokens
 * apart (dst_token_stride at least (n_heads - 1) * dst_head_stride + head_dim);
 * dst does not overlap q; window, sinks and max_kv in [0, 2^30]; n_heads and
 * n_seqs at most 65535; n_tokens at most 2^23, its product with
 * n_heads / n_kv_heads at most 2^30; n_seqs * n_kv_heads * ceil(max_q * n_heads
 * / n_kv_heads / R) at most 2^23, R the 16 to 128 rows of a workgroup that the
 * sizes give.  Deterministic.  The workspace is scratch: its contents do not
 * matter before the call, and it serves one call at a time.
 */
size_t hip_qmm_attn_paged_workspace_size(const hip_qmm_kv_cache *cache, int64_t n_heads, int64_t n_seqs,
                                         int64_t n_tokens, int64_t max_q, int64_t max_kv, int64_t window,
                                         int64_t sinks);
int hip_qmm_attn_paged(const hip_qmm_kv_cache *cache, const float *q, int64_t n_heads, int64_t q_token_stride,
                       int64_t q_head_stride, const int32_t *q_starts, int64_t n_seqs, int64_t n_tokens,
                       int64_t max_q, const int32_t *page_table, int64_t table_stride, const int32_t *kv_lens,
                       int64_t max_kv, float scale, int64_t window, int64_t sinks, float *dst,
                       int64_t dst_token_stride, int64_t dst_head_stride, void *workspace, size_t workspace_size,
                       void *stream);

/* What hip_qmm_attn_paged runs for these sizes, for measurement and tests:
 * the rows (query tokens x heads of a key-value head) of a workgroup, 16 or 32
 * in the few-row kernel and 64 or 128 in the many-row one, or 0 where the call
 * would be refused or empty; *splits, if not NULL (host), the most workgroups
 * that share a row's tokens. */
int hip_qmm_attn_paged_rows(const hip_qmm_kv_cache *cache, int64_t n_heads, int64_t n_seqs, int64_t n_tokens,
                            int64_t max_q, int64_t max_kv, int64_t window, int64_t sinks, int *splits);

/*
 * Copies pages inside the cache, keys and values: of page src[i] the first
 * n_tokens[i] tokens (NULL: all; values are cut to the page) into page dst[i], the rest
 * of which keeps its contents; i < n_copies.  A pair with a page outside the cache is
 * skipped.  No page may be the destination of two copies, or source and
 * destination.  A fork copies the partly filled last page and shares the
 * others in its row of the page table.
 */
int hip_qmm_kv_copy_pages(const hip_qmm_kv_cache *cache, const int32_t *src, const int32_t *dst,
                          const int32_t *n_tokens, int64_t n_copies, void *stream);

/*
 * Moves the pages in use to the front of the pool.  In use are the pages (in
 * [0, n_pages)) of the first ceil(kv_lens[s] / page_size) entries of each of
 * the n_seqs rows of page_table; rows may share pages.  With n_live of them,
 * the k-th page in use at or above n_live, ascending, moves to the k-th unused
 * page below n_live; table_out (n_seqs rows, its own stride, at least as wide;
 * page_table itself with the same stride, or apart from it) receives
 * page_table's table_width entries with the new numbers, -1 for those not in
 * use, and *n_live (apart from the others) the count: the pages from there on
 * are free.  A freed sequence has length 0.  All on the device, with no host
 * synchronization.  n_pages at most 2^20; the workspace is scratch.
 */
size_t hip_qmm_kv_compact_workspace_size(const hip_qmm_kv_cache *cache);
int hip_qmm_kv_compact(const hip_qmm_kv_cache *cache, const int32_t *page_table, int64_t table_stride,
                       int64_t table_width, const int32_t *kv_lens, int64_t n_seqs, int32_t *table_out,
                       int64_t out_stride, int32_t *n_live, void *workspace, size_t workspace_size, void *stream);

#ifdef __cplusplus
}
#endif

#endif /* GGML_HIP_ATTN_H */
