// kv_cache.h -- the paged key-value cache as the kernels see it, and the
// checks its entry points share (rope.hip, attn.hip, kv_pages.hip).
#pragma once

#include <hip/hip_fp16.h>
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "../../include/ggml_hip_attn.h"

namespace kvc {

struct Cache {
    uint16_t *k, *v;
    int64_t page_stride, head_stride, token_stride;  // elements
    int32_t n_pages, page_shift, n_kv_heads, head_dim;
};

// The host structure's check and its device form.
inline bool take(const hip_qmm_kv_cache *c, Cache *out) {
    if (!c || !c->k || !c->v) return false;
    if (c->type != HIP_QMM_TYPE_F16 && c->type != HIP_QMM_TYPE_BF16) return false;
    const int64_t D = c->head_dim, P = c->page_size, H = c->n_kv_heads;
    if (D < 8 || D > 256 || D % 8 || P < 16 || P > 65536 || (P & (P - 1)) || H < 1 || H > 65535) return false;
    if (c->n_pages < 1 || c->n_pages > INT32_MAX / P) return false;
    if (((uintptr_t)c->k | (uintptr_t)c->v) & 15) return false;
    const int64_t lim = (int64_t)1 << 40;
    if (c->page_stride < 0 || c->head_stride < 0 || c->token_stride < 0 || c->page_stride > lim ||
        c->head_stride > lim || c->token_stride > (1 << 27) || ((c->page_stride | c->head_stride | c->token_stride) & 7))
        return false;
    if (c->page_stride > INT64_MAX / 4 / c->n_pages) return false;
    // Either order of heads and tokens inside a page, nothing overlapping.
    const bool heads_out = c->token_stride >= D && (H == 1 || c->head_stride >= (P - 1) * c->token_stride + D);
    const bool tokens_out = (H == 1 || c->head_stride >= D) && c->token_stride >= (H - 1) * c->head_stride + D;
    if (!heads_out && !tokens_out) return false;
    if (c->n_pages > 1 && c->page_stride < (H - 1) * c->head_stride + (P - 1) * c->token_stride + D) return false;
    out->k = (uint16_t *)c->k;
    out->v = (uint16_t *)c->v;
    out->page_stride = c->page_stride;
    out->head_stride = c->head_stride;
    out->token_stride = c->token_stride;
    out->n_pages = (int32_t)c->n_pages;
    out->page_shift = __builtin_ctz((unsigned)P);
    out->n_kv_heads = (int32_t)H;
    out->head_dim = (int32_t)D;
    return true;
}

// f32 to the cache's 16 bits, to nearest even.  The empty statement keeps the
// f32 value: without it a product before the conversion becomes one mixed
// operation that rounds to f16 directly, and the stored key is no longer the
// rounding of what hip_qmm_rope_f32 gives.
template <bool BF16>
__device__ __forceinline__ uint16_t to16(float x) {
    asm("" : "+v"(x));
    if constexpr (BF16)
        return __builtin_bit_cast(uint16_t, (__bf16)x);
    else
        return __builtin_bit_cast(uint16_t, (_Float16)x);
}

template <bool BF16>
__device__ __forceinline__ float from16(uint16_t b) {
    if constexpr (BF16)
        return __uint_as_float((uint32_t)b << 16);
    else
        return (float)__builtin_bit_cast(_Float16, b);
}

}  // namespace kvc
