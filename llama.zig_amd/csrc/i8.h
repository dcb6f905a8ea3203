// i8.h -- what the sources of the 8-bit integer products share (i8_quantize.hip,
// i8_few.hip, i8_tile.hip, i8_api.hip).
#pragma once

#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

#include "../../include/ggml_hip_moe.h"

namespace i8 {

typedef int v4i __attribute__((ext_vector_type(4)));

constexpr int64_t MAX_K = 131071;         // 128 * 128 * K fits 31 bits
constexpr int64_t MAX_ROWS = 1 << 22;         // weight rows, columns, (token, slot) pairs
constexpr int64_t MAX_RESULTS = (int64_t)1 << 38;  // values of a result
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

// A row's largest magnitude, as the bits of an f32: integers compare as magnitudes do, and a NaN is above infinity.
__device__ __forceinline__ uint32_t magnitude(float x) { return __float_as_uint(x) & 0x7fffffffu; }

// Four values that need not be aligned to more than one: nor need a load of 16 bytes.
__device__ __forceinline__ float4 four_at(const float *x) {
    typedef float v4f __attribute__((ext_vector_type(4), aligned(4)));
    const v4f v = *reinterpret_cast<const v4f *>(x);
    return make_float4(v[0], v[1], v[2], v[3]);
}

// What a row's values are divided by.
struct Scale {
    float value;    // to be stored: NaN for a row that is not finite
    float divisor;
    float inverse;  // NaN where it might be no normal number, so that all values are divided
    bool usable;    // else all values are 0

    explicit __device__ __forceinline__ Scale(uint32_t most) {
        const bool finite = most < 0x7f800000u;
        divisor = __uint_as_float(most) * (1.0f / 127.0f);
        usable = finite && divisor > 0.0f;
        value = finite ? divisor : __uint_as_float(0x7fc00000u);
        inverse = divisor > 0x1p-120f && divisor < 0x1p120f ? 1.0f / divisor : __uint_as_float(0x7fc00000u);
    }

    // The quotient in IEEE arithmetic, to the nearest integer, half to even, at most 127.
    __device__ __forceinline__ int divided(float x) const {
        return usable ? (int)fminf(fmaxf(rintf(x / divisor), -127.0f), 127.0f) : 0;
    }

    // Four values, a byte each.  x * inverse is within 2^-15 of the quotient (which is below 128, and both roundings are
    // within 2^-23 of it), so a division decides only where a border between two integers is nearer than 2^-12.  Adding
    // 1.5 * 2^23 leaves the nearest integer in the lowest byte, in two's complement.
    __device__ __forceinline__ uint32_t four(float4 x) const {
        constexpr float ROUND = 0x1.8p23f;
        const float a = fmaf(x.x, inverse, ROUND), b = fmaf(x.y, inverse, ROUND), c = fmaf(x.z, inverse, ROUND),
                    d = fmaf(x.w, inverse, ROUND);
        const float away = fmaxf(fmaxf(fabsf(fmaf(x.x, inverse, ROUND - a)), fabsf(fmaf(x.y, inverse, ROUND - b))),
                                 fmaxf(fabsf(fmaf(x.z, inverse, ROUND - c)), fabsf(fmaf(x.w, inverse, ROUND - d))));
        if (inverse == inverse && away < 0.5f - 0x1p-12f) {
            const uint32_t low = __builtin_amdgcn_perm(__float_as_uint(b), __float_as_uint(a), 0x0c0c0400u);
            const uint32_t high = __builtin_amdgcn_perm(__float_as_uint(d), __float_as_uint(c), 0x04000c0cu);
            return low | high;
        }
        return (divided(x.x) & 255) | (divided(x.y) & 255) << 8 | (divided(x.z) & 255) << 16 | (uint32_t)divided(x.w) << 24;
    }
};

// A sum times its two scales: three f32 roundings (the sum's and two products'), of mantissas alone, so that no
// product leaves the range of f32 unless the result does.  The last product is exact in f64 and rounded once, to the
// fewer bits that a subnormal result has too (f32 would round it to 24 bits before).
__device__ __forceinline__ float scaled(int sum, float x_scale, float w_scale) {
    const float product = (float)sum * __builtin_amdgcn_frexp_mantf(x_scale);
    return (float)ldexp((double)product * (double)__builtin_amdgcn_frexp_mantf(w_scale),
                        __builtin_amdgcn_frexp_expf(x_scale) + __builtin_amdgcn_frexp_expf(w_scale));
}

// Scales with which the products may be taken as they are, with the same bits.
__device__ __forceinline__ bool moderate(float scale) {
    const float s = fabsf(scale);
    return s == 0.0f || (s > 0x1p-60f && s < 0x1p60f);
}

constexpr int PAIR_CHUNK = 4096;  // (token, slot) pairs of a grouping workgroup

// The grouping's tables: see Product; counts and places are its own.
struct Groups {
    int32_t *col_src, *col_dst, *tiles, *n_tiles, *counts;
    uint16_t *places;
};

// i8_quantize.hip
int quantize(const float *x, int64_t K, int64_t n_rows, int64_t x_stride, int8_t *q, int64_t q_stride, float *scale,
             hipStream_t s);
// The tables; and, in the same launch, n_rows f32 rows of K at x as 8-bit ones (x NULL: none).
int group(const int32_t *ids, int64_t ids_stride, int n_pairs, int n_ids, int n_as, int per_slot, int bn, const Groups &to,
          float *dst, int64_t dst_stride, int64_t nrows, const float *x, int64_t K, int64_t n_rows, int64_t x_stride,
          int8_t *q, int64_t q_stride, float *scale, hipStream_t s);

// i8_few.hip: how few columns are taken, from the sizes alone.
enum FewMode { QUANTIZE, RESIDENT, THROUGH };  // f32 columns quantized in LDS; 8-bit ones in LDS; through the ring
struct FewPlan {
    FewMode mode;
    int nt, depth, rows;     // column tiles, items ahead, weight rows of a workgroup
    int columns, staged;     // in LDS at once; of f32
    int bytes;               // of LDS; 0: not taken
};
FewPlan few_plan(bool f32, int64_t K, int64_t nrows, int64_t ncols);
FewPlan few_pairs_plan(bool f32, int64_t K, int64_t nrows, int64_t n_as, int64_t n_tokens, int64_t n_ids);
// p.x is f32 where the plan's mode is QUANTIZE
int few_product(const Product &p, const FewPlan &plan, hipStream_t s);
int few_pairs(const Product &p, const FewPlan &plan, const int32_t *ids, int64_t ids_stride, int n_pairs, int n_ids, int n_as,
              int per_slot, hipStream_t s);

// i8_tile.hip: tiles of TM weight rows and TN columns.
enum TileForm { TILE_64x64, TILE_128x64, TILE_128x128, TILE_128x128_DEEP, TILE_256x256 };
TileForm tile_form(int64_t nrows, int64_t ncols);                   // dense
TileForm tile_form_grouped(int64_t K, int64_t nrows, int64_t n_as, int64_t n_pairs);  // by experts
int tile_columns(TileForm form);
int tile_product(const Product &p, TileForm form, int64_t max_tiles, hipStream_t s);

}  // namespace i8
