// i8_api.hip -- the entry points of the 8-bit products: their checks, their
// workspaces, and which kernel runs.
#include <algorithm>

#include "i8.h"

using namespace i8;

namespace {

size_t a256(size_t n) { return (n + 255) / 256 * 256; }

bool sizes_ok(int64_t K, int64_t nrows) { return K >= 1 && K <= MAX_K && nrows >= 1 && nrows <= MAX_ROWS; }

// Quantized tokens in the workspace: rows of whole 128 bytes.
int64_t token_stride(int64_t K) { return (K + 127) / 128 * 128; }

struct Tokens {
    size_t q, scale, end;
};

Tokens tokens_at(size_t at, int64_t K, int64_t n) {
    Tokens t;
    t.q = at;
    t.scale = a256(t.q + (size_t)(n * token_stride(K)));
    t.end = a256(t.scale + (size_t)n * 4);
    return t;
}

struct Grouped {
    size_t src, dst, tiles, n_tiles, counts, places, end;
    TileForm form;
    int64_t max_tiles;
};

Grouped grouped_at(size_t at, int64_t K, int64_t nrows, int64_t n_as, int64_t pairs) {
    Grouped g;
    g.form = tile_form_grouped(K, nrows, n_as, pairs);
    g.max_tiles = pairs / tile_columns(g.form) + std::min(pairs, n_as);
    g.src = at;
    g.dst = a256(g.src + (size_t)pairs * 4);
    g.tiles = a256(g.dst + (size_t)pairs * 4);
    g.n_tiles = a256(g.tiles + (size_t)g.max_tiles * 16);
    g.counts = a256(g.n_tiles + 4);
    g.places = a256(g.counts + (size_t)((pairs + PAIR_CHUNK - 1) / PAIR_CHUNK * n_as) * 4);
    g.end = a256(g.places + (size_t)pairs * 2);
    return g;
}

bool operand_ok(const void *p, int64_t stride, int64_t K, bool bytes) {
    if (!p || stride < K || stride > MAX_STRIDE) return false;
    return bytes ? !((uintptr_t)p % 16 || stride % 16) : !((uintptr_t)p % 4);
}

// Tensors of 4-byte values.
bool words_ok(const void *p) { return p && !((uintptr_t)p % 4); }

bool workspace_ok(const void *ws, size_t have, size_t need) {
    return need == 0 || (ws && !((uintptr_t)ws % 256) && have >= need);
}

// p with its columns as they will be in the workspace.
Product quantized_tokens(Product p, const Tokens &t, void *workspace) {
    p.x = (const int8_t *)workspace + t.q, p.x_scale = (const float *)((uint8_t *)workspace + t.scale);
    p.x_stride = token_stride(p.K);
    return p;
}

}  // namespace

extern "C" size_t hip_qmm_mul_mat_i8_workspace_size(int64_t K, int64_t nrows, int64_t ncols, int quantized) {
    if (!sizes_ok(K, nrows) || ncols < 1 || ncols > MAX_ROWS || quantized || few_plan(true, K, nrows, ncols).bytes) return 0;
    return tokens_at(0, K, ncols).end;
}

extern "C" int hip_qmm_mul_mat_i8(const int8_t *w, const float *w_scale, int64_t K, int64_t nrows, int64_t w_stride,
                                  const void *x, const float *x_scale, int64_t ncols, int64_t x_stride, float *dst,
                                  int64_t dst_stride, void *workspace, size_t workspace_size, void *stream) {
    if (!sizes_ok(K, nrows) || ncols < 0 || ncols > MAX_ROWS) return (int)hipErrorInvalidValue;
    if (ncols == 0) return 0;
    if (nrows > MAX_RESULTS / ncols) return (int)hipErrorInvalidValue;
    if (!words_ok(w_scale) || !words_ok(dst) || (x_scale && !words_ok(x_scale)) || dst_stride < nrows ||
        dst_stride > MAX_STRIDE || !operand_ok(w, w_stride, K, true) || !operand_ok(x, x_stride, K, x_scale != nullptr) ||
        !workspace_ok(workspace, workspace_size, hip_qmm_mul_mat_i8_workspace_size(K, nrows, ncols, x_scale != nullptr)))
        return (int)hipErrorInvalidValue;
    hipStream_t s = (hipStream_t)stream;
    Product p = {};
    p.w = w, p.w_scale = w_scale, p.w_stride = w_stride;
    p.dst = dst, p.dst_stride = dst_stride;
    p.K = (int)K, p.nrows = (int)nrows, p.ncols = (int)ncols;
    p.x = (const int8_t *)x, p.x_scale = x_scale, p.x_stride = x_stride;
    if (!x_scale) {
        const FewPlan plan = few_plan(true, K, nrows, ncols);
        if (plan.bytes) return few_product(p, plan, s);
        p = quantized_tokens(p, tokens_at(0, K, ncols), workspace);
        if (int e = quantize((const float *)x, K, ncols, x_stride, (int8_t *)p.x, p.x_stride, (float *)p.x_scale, s)) return e;
    }
    const FewPlan plan = few_plan(false, K, nrows, ncols);
    // Many rows and over 16 columns: tiles, whose workgroups share the columns (14336 x 4096 by 32: 15 us, 19 us).
    if (plan.bytes && (ncols <= 16 || plan.mode == RESIDENT || nrows < 8192)) return few_product(p, plan, s);
    const TileForm form = tile_form(nrows, ncols);
    const int bn = tile_columns(form);
    return tile_product(p, form, (ncols + bn - 1) / bn, s);
}

extern "C" size_t hip_qmm_mul_mat_id_i8_workspace_size(int64_t K, int64_t nrows, int64_t n_as, int64_t ne11,
                                                       int64_t n_tokens, int64_t n_ids, int quantized) {
    if (!sizes_ok(K, nrows) || n_as < 1 || n_as > MAX_EXPERTS || n_tokens < 1 || n_ids < 1 || n_ids > MAX_ROWS ||
        n_tokens > MAX_ROWS / n_ids || (ne11 != 1 && ne11 != n_ids))
        return 0;
    const bool few = few_pairs_plan(false, K, nrows, n_as, n_tokens, n_ids).bytes != 0;  // no tables
    if (!quantized && few_pairs_plan(true, K, nrows, n_as, n_tokens, n_ids).bytes) return 0;
    if (few) return quantized ? 0 : tokens_at(0, K, n_tokens * ne11).end;
    return grouped_at(quantized ? 0 : tokens_at(0, K, n_tokens * ne11).end, K, nrows, n_as, n_tokens * n_ids).end;
}

extern "C" int hip_qmm_mul_mat_id_i8(const int8_t *w, const float *w_scale, int64_t K, int64_t nrows, int64_t w_stride,
                                     int64_t expert_stride, int64_t n_as, const void *x, const float *x_scale,
                                     int64_t ne11, int64_t n_tokens, int64_t x_stride, const int32_t *ids,
                                     int64_t n_ids, int64_t ids_stride, float *dst, int64_t dst_stride,
                                     void *workspace, size_t workspace_size, void *stream) {
    if (!sizes_ok(K, nrows) || n_as < 1 || n_as > MAX_EXPERTS || n_tokens < 0 || n_ids < 0 || n_ids > MAX_ROWS ||
        n_tokens > MAX_ROWS || (n_ids > 0 && n_tokens > MAX_ROWS / n_ids) || (ne11 != 1 && ne11 != n_ids))
        return (int)hipErrorInvalidValue;
    if (n_tokens == 0 || n_ids == 0) return 0;
    if (nrows > MAX_RESULTS / (n_tokens * n_ids)) return (int)hipErrorInvalidValue;
    const bool quantized = x_scale != nullptr;
    if (!words_ok(w_scale) || !words_ok(dst) || !words_ok(ids) || (quantized && !words_ok(x_scale)) || ids_stride < n_ids ||
        ids_stride > MAX_STRIDE || dst_stride < nrows ||
        dst_stride > MAX_STRIDE || !operand_ok(w, w_stride, K, true) || expert_stride % 16 ||
        expert_stride < (nrows - 1) * w_stride + K || expert_stride > MAX_STRIDE ||
        !operand_ok(x, x_stride, K, quantized) ||
        !workspace_ok(workspace, workspace_size,
                      hip_qmm_mul_mat_id_i8_workspace_size(K, nrows, n_as, ne11, n_tokens, n_ids, quantized)))
        return (int)hipErrorInvalidValue;
    hipStream_t s = (hipStream_t)stream;
    uint8_t *ws = (uint8_t *)workspace;
    const Tokens t = tokens_at(0, K, n_tokens * ne11);
    const Grouped g = grouped_at(quantized ? 0 : t.end, K, nrows, n_as, n_tokens * n_ids);
    Product p = {};
    p.w = w, p.w_scale = w_scale, p.w_stride = w_stride, p.expert_stride = expert_stride;
    p.dst = dst, p.dst_stride = dst_stride;
    p.K = (int)K, p.nrows = (int)nrows;
    p.x = (const int8_t *)x, p.x_scale = x_scale, p.x_stride = x_stride;
    const int pairs = (int)(n_tokens * n_ids);
    if (!quantized) {
        const FewPlan plan = few_pairs_plan(true, K, nrows, n_as, n_tokens, n_ids);
        if (plan.bytes) return few_pairs(p, plan, ids, ids_stride, pairs, (int)n_ids, (int)n_as, ne11 > 1, s);
        p = quantized_tokens(p, t, workspace);
    }
    const float *xf = quantized ? nullptr : (const float *)x;
    int8_t *q = (int8_t *)p.x;
    float *scale = (float *)p.x_scale;
    const FewPlan plan = few_pairs_plan(false, K, nrows, n_as, n_tokens, n_ids);
    if (plan.bytes) {
        if (xf)
            if (int e = quantize(xf, K, n_tokens * ne11, x_stride, q, p.x_stride, scale, s)) return e;
        return few_pairs(p, plan, ids, ids_stride, pairs, (int)n_ids, (int)n_as, ne11 > 1, s);
    }
    const Groups to = {(int32_t *)(ws + g.src), (int32_t *)(ws + g.dst), (int32_t *)(ws + g.tiles),
                       (int32_t *)(ws + g.n_tiles), (int32_t *)(ws + g.counts), (uint16_t *)(ws + g.places)};
    if (int e = group(ids, ids_stride, pairs, (int)n_ids, (int)n_as, ne11 > 1, tile_columns(g.form), to, dst, dst_stride,
                      nrows, xf, K, n_tokens * ne11, x_stride, q, p.x_stride, scale, s))
        return e;
    p.tiles = to.tiles, p.n_tiles = to.n_tiles, p.col_src = to.col_src, p.col_dst = to.col_dst;
    return tile_product(p, g.form, g.max_tiles, s);
}
