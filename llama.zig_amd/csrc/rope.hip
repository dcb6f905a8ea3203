// rope.hip -- rotary positions, and the store of rotated keys and plain
// values into the paged cache.
//
// The turn of pair i at position p is p * step_i in units of 2^-64 turns,
// with whole turns dropped by the 64-bit wrap: exact, where an f32 angle
// p * f_i loses p * 2^-24 radians.  Its 64 bits, taken as signed, become the
// argument of sincospi in [-1, 1), so that small angles keep their relative
// precision too.
//
// HBM bound: one pass, 16-byte loads and stores.  A workgroup takes rows
// (heads of q, then k, then v) of one token; a thread eight elements of one
// row: four pairs, whose turns it computes itself (four sincospi hide behind
// the loads).
#include <math.h>

#include "kv_cache.h"

using namespace kvc;

namespace {

constexpr int THREADS = 256;

struct Rows {
    const float *src;
    int64_t token, head;  // strides
    int n;
};

struct RopeArgs {
    Rows q, k, v;  // k and v empty without a cache
    float *dst;
    int64_t dst_token, dst_head;
    const int32_t *pos, *slots;
    const int64_t *steps;
    int head_dim, half;  // half = n_dims / 2
    float mscale;
    Cache cache;
};

__device__ __forceinline__ void turn(const RopeArgs &a, int64_t pos, int i, float *c, float *s) {
    const uint64_t phase = (uint64_t)pos * (uint64_t)a.steps[i];
    sincospif((float)(int64_t)phase * 0x1p-63f, s, c);
    *c *= a.mscale;
    *s *= a.mscale;
}

// Element e of `half` pairs' first or second member in its layout.
template <int LAYOUT>
__device__ __forceinline__ int first_of(int i) { return LAYOUT == HIP_QMM_ROPE_HALF ? i : 2 * i; }
template <int LAYOUT>
__device__ __forceinline__ int second_of(int i, int half) { return LAYOUT == HIP_QMM_ROPE_HALF ? i + half : 2 * i + 1; }

template <bool BF16>
__device__ __forceinline__ void put(float *d, float x) { *d = x; }
template <bool BF16>
__device__ __forceinline__ void put(uint16_t *d, float x) { *d = to16<BF16>(x); }

// Any head_dim, n_dims, alignment: one pair or one plain element per thread
// and step.
template <int LAYOUT, bool BF16, class Out>
__device__ __forceinline__ void row_any(const RopeArgs &a, const float *x, Out *d, int64_t pos, bool rotate, int lane,
                                        int lanes) {
    const int half = rotate ? a.half : 0;
    for (int i = lane; i < half; i += lanes) {
        float c, s;
        turn(a, pos, i, &c, &s);
        const int e = first_of<LAYOUT>(i), f = second_of<LAYOUT>(i, half);
        const float p = x[e], q = x[f];
        put<BF16>(d + e, fmaf(p, c, -(q * s)));
        put<BF16>(d + f, fmaf(p, s, q * c));
    }
    for (int e = 2 * half + lane; e < a.head_dim; e += lanes) put<BF16>(d + e, x[e]);
}

template <int LAYOUT, bool BF16>
__global__ __launch_bounds__(THREADS) void rope_kernel(RopeArgs a) {
    const int64_t t = blockIdx.x;
    const int64_t pos = a.pos[t];
    const int rows = a.q.n + a.k.n + a.v.n, wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    for (int r = blockIdx.y * (THREADS / 64) + wave; r < rows; r += gridDim.y * (THREADS / 64)) {
        if (r < a.q.n) {
            row_any<LAYOUT, BF16>(a, a.q.src + t * a.q.token + r * a.q.head, a.dst + t * a.dst_token + r * a.dst_head,
                                  pos, true, lane, 64);
            continue;
        }
        const int slot = a.slots[t];
        if (slot < 0 || (slot >> a.cache.page_shift) >= a.cache.n_pages) continue;
        const bool key = r < a.q.n + a.k.n;
        const int h = key ? r - a.q.n : r - a.q.n - a.k.n;
        const Rows &in = key ? a.k : a.v;
        uint16_t *d = (key ? a.cache.k : a.cache.v) + (int64_t)(slot >> a.cache.page_shift) * a.cache.page_stride +
                      (int64_t)(slot & ((1 << a.cache.page_shift) - 1)) * a.cache.token_stride + h * a.cache.head_stride;
        row_any<LAYOUT, BF16>(a, in.src + t * in.token + h * in.head, d, pos, key, lane, 64);
    }
}

template <int LAYOUT, bool BF16>
int launch(const RopeArgs &a, int64_t n_tokens, hipStream_t s) {
    const int rows = a.q.n + a.k.n + a.v.n;
    const dim3 grid((unsigned)n_tokens, (unsigned)((rows + THREADS / 64 - 1) / (THREADS / 64)));
    hipLaunchKernelGGL((rope_kernel<LAYOUT, BF16>), grid, dim3(THREADS), 0, s, a);
    return (int)hipGetLastError();
}

int launch_any(const RopeArgs &a, int64_t n_tokens, int layout, bool bf16, void *stream) {
    hipStream_t s = (hipStream_t)stream;
    if (layout == HIP_QMM_ROPE_HALF)
        return bf16 ? launch<HIP_QMM_ROPE_HALF, true>(a, n_tokens, s) : launch<HIP_QMM_ROPE_HALF, false>(a, n_tokens, s);
    return bf16 ? launch<HIP_QMM_ROPE_INTERLEAVED, true>(a, n_tokens, s)
                : launch<HIP_QMM_ROPE_INTERLEAVED, false>(a, n_tokens, s);
}

bool fine_strides(int64_t n_tokens, int64_t n_heads, int64_t D, int64_t token, int64_t head) {
    const int64_t lim = (int64_t)1 << 40;
    return token >= 0 && head >= 0 && token < lim && head < lim && (n_heads < 2 || head >= D) &&
           (n_tokens < 2 || n_heads < 1 || token >= (n_heads - 1) * head + D || (head >= (n_tokens - 1) * token + D && token >= D));
}

bool fine_shape(int64_t n_tokens, int64_t n_heads, int64_t head_dim, int n_dims, int layout, float mscale) {
    return n_tokens >= 0 && n_tokens <= ((int64_t)1 << 23) && n_heads >= 0 && n_heads <= 65535 && head_dim >= 1 &&
           head_dim <= 1024 && n_dims >= 2 && n_dims <= 256 && n_dims <= head_dim && !(n_dims & 1) &&
           (layout == HIP_QMM_ROPE_HALF || layout == HIP_QMM_ROPE_INTERLEAVED) && mscale == mscale;
}

}  // namespace

extern "C" int hip_qmm_rope_steps(int n_dims, double freq_base, double freq_scale, double ext_factor,
                                  double attn_factor, double beta_fast, double beta_slow, int64_t n_ctx_orig,
                                  const float *freq_factors, int64_t *steps, float *mscale) {
    if (n_dims < 2 || n_dims > 256 || (n_dims & 1) || !steps || !mscale) return (int)hipErrorInvalidValue;
    if (!(freq_base > 1.0) || !(freq_scale > 0.0) || !(ext_factor >= 0.0) || !isfinite(freq_base) ||
        !isfinite(freq_scale) || !isfinite(ext_factor) || !isfinite(attn_factor))
        return (int)hipErrorInvalidValue;
    if (ext_factor > 0.0 && (!(beta_fast > 0.0) || !(beta_slow > 0.0) || n_ctx_orig < 1)) return (int)hipErrorInvalidValue;
    const double two_pi = 6.283185307179586476925286766559;
    double low = 0.0, high = 0.0;
    if (ext_factor > 0.0) {
        // The pair that turns `beta` times over n_ctx_orig positions: f = 2 pi beta / n_ctx_orig solved for i.
        const double per = n_dims / (2.0 * log(freq_base));
        low = fmax(0.0, floor(per * log((double)n_ctx_orig / (beta_fast * two_pi))));
        high = fmin(n_dims - 1.0, ceil(per * log((double)n_ctx_orig / (beta_slow * two_pi))));
    }
    for (int i = 0; i < n_dims / 2; ++i) {
        const double factor = freq_factors ? (double)freq_factors[i] : 1.0;
        if (!(factor > 0.0) || !isfinite(factor)) return (int)hipErrorInvalidValue;
        const double f = pow(freq_base, -2.0 * i / n_dims) / factor;
        double g = f * freq_scale;
        if (ext_factor > 0.0) {
            const double keep = (1.0 - fmin(1.0, fmax(0.0, (i - low) / fmax(0.001, high - low)))) * ext_factor;
            g = g * (1.0 - keep) + f * keep;
        }
        double turns = g / two_pi;
        turns -= floor(turns);
        if (turns >= 0.5) turns -= 1.0;
        const double whole = rint(turns * 0x1p64);  // in [-2^63, 2^63]
        steps[i] = whole >= 0x1p63 ? INT64_MIN : (int64_t)whole;
    }
    *mscale = (float)(attn_factor * (ext_factor > 0.0 ? 1.0 + 0.1 * log(1.0 / freq_scale) : 1.0));
    return 0;
}

extern "C" int hip_qmm_rope_f32(const float *x, int64_t n_tokens, int64_t n_heads, int64_t head_dim,
                                int64_t x_token_stride, int64_t x_head_stride, const int32_t *pos,
                                const int64_t *steps, int n_dims, int layout, float mscale, float *dst,
                                int64_t dst_token_stride, int64_t dst_head_stride, void *stream) {
    if (!fine_shape(n_tokens, n_heads, head_dim, n_dims, layout, mscale) || !x || !pos || !steps || !dst ||
        !fine_strides(n_tokens, n_heads, head_dim, x_token_stride, x_head_stride) ||
        !fine_strides(n_tokens, n_heads, head_dim, dst_token_stride, dst_head_stride))
        return (int)hipErrorInvalidValue;
    if (n_tokens == 0 || n_heads == 0) return 0;
    RopeArgs a = {};
    a.q = {x, x_token_stride, x_head_stride, (int)n_heads};
    a.dst = dst;
    a.dst_token = dst_token_stride;
    a.dst_head = dst_head_stride;
    a.pos = pos;
    a.steps = steps;
    a.head_dim = (int)head_dim;
    a.half = n_dims / 2;
    a.mscale = mscale;
    return launch_any(a, n_tokens, layout, false, stream);
}

extern "C" int hip_qmm_rope_kv_store(const float *q, int64_t n_heads, int64_t q_token_stride, int64_t q_head_stride,
                                     const float *k, const float *v, int64_t kv_token_stride, int64_t kv_head_stride,
                                     int64_t n_tokens, const int32_t *pos, const int64_t *steps, int n_dims,
                                     int layout, float mscale, float *q_dst, int64_t dst_token_stride,
                                     int64_t dst_head_stride, const hip_qmm_kv_cache *cache, const int32_t *slots,
                                     void *stream) {
    RopeArgs a = {};
    if (!take(cache, &a.cache)) return (int)hipErrorInvalidValue;
    const int64_t D = a.cache.head_dim, H = a.cache.n_kv_heads;
    if (!fine_shape(n_tokens, n_heads, D, n_dims, layout, mscale) || !k || !v || !pos || !steps || !slots ||
        !fine_strides(n_tokens, H, D, kv_token_stride, kv_head_stride))
        return (int)hipErrorInvalidValue;
    if (n_heads > 0 && (!q || !q_dst || !fine_strides(n_tokens, n_heads, D, q_token_stride, q_head_stride) ||
                        !fine_strides(n_tokens, n_heads, D, dst_token_stride, dst_head_stride)))
        return (int)hipErrorInvalidValue;
    if (n_tokens == 0) return 0;
    a.q = {q, q_token_stride, q_head_stride, (int)n_heads};
    a.k = {k, kv_token_stride, kv_head_stride, (int)H};
    a.v = {v, kv_token_stride, kv_head_stride, (int)H};
    a.dst = q_dst;
    a.dst_token = dst_token_stride;
    a.dst_head = dst_head_stride;
    a.pos = pos;
    a.slots = slots;
    a.steps = steps;
    a.head_dim = (int)D;
    a.half = n_dims / 2;
    a.mscale = mscale;
    return launch_any(a, n_tokens, layout, cache->type == HIP_QMM_TYPE_BF16, stream);
}
