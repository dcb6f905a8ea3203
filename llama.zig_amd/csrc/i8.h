// i8.h -- what the sources of the 8-bit integer products share (i8_quantize.hip,
// i8_stream.hip, i8_api.hip).
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "../../include/ggml_hip_moe.h"

namespace i8 {

typedef int v4i __attribute__((ext_vector_type(4)));

constexpr int64_t MAX_K = 131071;         // 128 * 128 * K fits 31 bits
constexpr int64_t MAX_ROWS = 1 << 22;         // weight rows, columns, (token, slot) pairs
constexpr int64_t MAX_EXPERTS = 1024;
constexpr int64_t MAX_STRIDE = (int64_t)1 << 40;

// A product, dense or by experts.  By experts column c stands at x row
// col_src[c] and dst row col_dst[c], and tile i = {expert, first column, end, 0}
// of tiles[0 .. *n_tiles).
struct Product {
    const int8_t *w;
    const float *w_scale;
    int64_t w_stride, expert_stride;
    const int8_t *x;
    const float *x_scale;
    int64_t x_stride;
    float *dst;
    int64_t dst_stride;
    const int32_t *tiles, *n_tiles, *col_src, *col_dst;  // NULL: dense
    int K, nrows, ncols;
};

// Bytes of a 16-byte chunk from `keep` on are cleared.
__device__ __forceinline__ v4i cut(v4i v, int keep) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int n = min(max(keep - 4 * i, 0), 4);
        v[i] = n == 4 ? v[i] : v[i] & ((1u << (8 * n)) - 1);
    }
    return v;
}

// A sum times its two scales, rounded to f32 once: in f32 either product could leave its range though the result
// does not, and f64 instructions are as fast here.
__device__ __forceinline__ float scaled(int sum, float x_scale, float w_scale) {
    return (float)((double)sum * (double)x_scale * (double)w_scale);
}

// i8_quantize.hip
int quantize(const float *x, int64_t K, int64_t n_rows, int64_t x_stride, int8_t *q, int64_t q_stride, float *scale,
             hipStream_t s);
int group(const int32_t *ids, int64_t ids_stride, int64_t n_tokens, int64_t n_ids, int64_t n_as, int64_t ne11, int bn,
          int32_t *col_src, int32_t *col_dst, int32_t *tiles, int32_t *n_tiles, float *dst, int64_t dst_stride,
          int64_t nrows, hipStream_t s);
// i8_stream.hip
int stream_product(const Product &p, int64_t max_tiles, int bn, hipStream_t s);

}  // namespace i8
