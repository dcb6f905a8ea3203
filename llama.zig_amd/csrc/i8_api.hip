// i8_api.hip -- the entry points of the 8-bit products: their checks, their
// workspaces, and which kernel runs.
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

// A tile's columns.
int columns(int64_t n) { return n <= 16 ? 16 : n <= 32 ? 32 : 64; }

struct Grouped {
    size_t src, dst, tiles, n_tiles, end;
    int bn;
    int64_t max_tiles;
};

Grouped grouped_at(size_t at, int64_t n_as, int64_t pairs) {
    Grouped g;
    g.bn = columns((pairs + n_as - 1) / n_as);
    g.max_tiles = pairs / g.bn + (pairs < n_as ? pairs : n_as);
    g.src = at;
    g.dst = a256(g.src + (size_t)pairs * 4);
    g.tiles = a256(g.dst + (size_t)pairs * 4);
    g.n_tiles = a256(g.tiles + (size_t)g.max_tiles * 16);
    g.end = a256(g.n_tiles + 4);
    return g;
}

bool operand_ok(const void *p, int64_t stride, int64_t K, bool bytes) {
    if (!p || stride < K || stride > MAX_STRIDE) return false;
    return bytes ? !((uintptr_t)p % 16 || stride % 16) : !((uintptr_t)p % 4);
}

bool workspace_ok(const void *ws, size_t have, size_t need) {
    return need == 0 || (ws && !((uintptr_t)ws % 256) && have >= need);
}

}  // namespace

extern "C" size_t hip_qmm_mul_mat_i8_workspace_size(int64_t K, int64_t nrows, int64_t ncols, int quantized) {
    if (!sizes_ok(K, nrows) || ncols < 1 || ncols > MAX_ROWS || quantized) return 0;
    return tokens_at(0, K, ncols).end;
}

extern "C" int hip_qmm_mul_mat_i8(const int8_t *w, const float *w_scale, int64_t K, int64_t nrows, int64_t w_stride,
                                  const void *x, const float *x_scale, int64_t ncols, int64_t x_stride, float *dst,
                                  int64_t dst_stride, void *workspace, size_t workspace_size, void *stream) {
    if (!sizes_ok(K, nrows) || ncols < 0 || ncols > MAX_ROWS) return (int)hipErrorInvalidValue;
    if (ncols == 0) return 0;
    if (!w_scale || !dst || dst_stride < nrows || dst_stride > MAX_STRIDE || !operand_ok(w, w_stride, K, true) ||
        !operand_ok(x, x_stride, K, x_scale != nullptr) ||
        !workspace_ok(workspace, workspace_size, hip_qmm_mul_mat_i8_workspace_size(K, nrows, ncols, x_scale != nullptr)))
        return (int)hipErrorInvalidValue;
    hipStream_t s = (hipStream_t)stream;
    Product p = {};
    p.w = w, p.w_scale = w_scale, p.w_stride = w_stride;
    p.dst = dst, p.dst_stride = dst_stride;
    p.K = (int)K, p.nrows = (int)nrows, p.ncols = (int)ncols;
    p.x = (const int8_t *)x, p.x_scale = x_scale, p.x_stride = x_stride;
    if (!x_scale) {
        uint8_t *ws = (uint8_t *)workspace;
        const Tokens t = tokens_at(0, K, ncols);
        const int64_t stride = token_stride(K);
        if (int e = quantize((const float *)x, K, ncols, x_stride, (int8_t *)(ws + t.q), stride, (float *)(ws + t.scale), s))
            return e;
        p.x = (const int8_t *)(ws + t.q), p.x_scale = (const float *)(ws + t.scale), p.x_stride = stride;
    }
    const int bn = columns(ncols);
    return stream_product(p, (ncols + bn - 1) / bn, bn, s);
}

extern "C" size_t hip_qmm_mul_mat_id_i8_workspace_size(int64_t K, int64_t nrows, int64_t n_as, int64_t ne11,
                                                       int64_t n_tokens, int64_t n_ids, int quantized) {
    if (!sizes_ok(K, nrows) || n_as < 1 || n_as > MAX_EXPERTS || n_tokens < 1 || n_ids < 1 || n_ids > MAX_ROWS ||
        n_tokens > MAX_ROWS / n_ids || (ne11 != 1 && ne11 != n_ids))
        return 0;
    return grouped_at(quantized ? 0 : tokens_at(0, K, n_tokens * ne11).end, n_as, n_tokens * n_ids).end;
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
    const bool quantized = x_scale != nullptr;
    if (!w_scale || !dst || !ids || ids_stride < n_ids || ids_stride > MAX_STRIDE || dst_stride < nrows ||
        dst_stride > MAX_STRIDE || !operand_ok(w, w_stride, K, true) || expert_stride % 16 ||
        expert_stride < (nrows - 1) * w_stride + K || expert_stride > MAX_STRIDE ||
        !operand_ok(x, x_stride, K, quantized) ||
        !workspace_ok(workspace, workspace_size,
                      hip_qmm_mul_mat_id_i8_workspace_size(K, nrows, n_as, ne11, n_tokens, n_ids, quantized)))
        return (int)hipErrorInvalidValue;
    hipStream_t s = (hipStream_t)stream;
    uint8_t *ws = (uint8_t *)workspace;
    const Tokens t = tokens_at(0, K, n_tokens * ne11);
    const Grouped g = grouped_at(quantized ? 0 : t.end, n_as, n_tokens * n_ids);
    Product p = {};
    p.w = w, p.w_scale = w_scale, p.w_stride = w_stride, p.expert_stride = expert_stride;
    p.dst = dst, p.dst_stride = dst_stride;
    p.K = (int)K, p.nrows = (int)nrows;
    p.x = (const int8_t *)x, p.x_scale = x_scale, p.x_stride = x_stride;
    if (!quantized) {
        const int64_t stride = token_stride(K);
        if (int e = quantize((const float *)x, K, n_tokens * ne11, x_stride, (int8_t *)(ws + t.q), stride,
                             (float *)(ws + t.scale), s))
            return e;
        p.x = (const int8_t *)(ws + t.q), p.x_scale = (const float *)(ws + t.scale), p.x_stride = stride;
    }
    int32_t *src = (int32_t *)(ws + g.src), *to = (int32_t *)(ws + g.dst);
    int32_t *tiles = (int32_t *)(ws + g.tiles), *n_tiles = (int32_t *)(ws + g.n_tiles);
    if (int e = group(ids, ids_stride, n_tokens, n_ids, n_as, ne11, g.bn, src, to, tiles, n_tiles, dst, dst_stride, nrows, s))
        return e;
    p.tiles = tiles, p.n_tiles = n_tiles, p.col_src = src, p.col_dst = to;
    return stream_product(p, g.max_tiles, g.bn, s);
}
