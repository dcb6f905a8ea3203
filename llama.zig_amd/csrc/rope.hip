// rope.hip -- rotary positions, and the store of rotated keys and plain
// values into the paged cache.
//
// The turn of pair i at position p is p * step_i in units of 2^-64 turns,
// with whole turns dropped by the 64-bit wrap: exact, where an f32 angle
// p * f_i loses p * 2^-24 radians.  Its 64 bits, taken as signed, become the
// argument of sincospi in [-1, 1), so that small angles keep their relative
// precision too.
//
// HBM bound: one pass, 16-byte loads.  A workgroup takes the rows (heads of q,
// then k, then v) of one token; a thread eight elements of a row, four pairs,
// and computes their turns once for all of its rows, while other workgroups
// load.  8192 tokens of 32 + 8 + 8 heads of 128 (369 MB): 69 us, 5.3 TB/s, what
// a large copy reaches on this card; one such token 2.5 us, a launch.
#include <math.h>

#include "kv_cache.h"

using namespace kvc;

namespace {

constexpr int THREADS = 256;
constexpr int64_t FEW_TOKENS = 512;

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

// One pair or one plain element per lane and step.
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

// Where row r (of q, then k, then v) of token t comes from, and where it goes:
// one of the two destinations, or none (false).
struct Place {
    const float *from;
    float *to;
    uint16_t *stored;
    bool rotate;
};

__device__ __forceinline__ bool place_of(const RopeArgs &a, int64_t t, int r, int slot, Place *p) {
    if (r < a.q.n) {
        *p = {a.q.src + t * a.q.token + r * a.q.head, a.dst + t * a.dst_token + r * a.dst_head, nullptr, true};
        return true;
    }
    if (slot < 0 || (slot >> a.cache.page_shift) >= a.cache.n_pages) return false;
    const bool key = r < a.q.n + a.k.n;
    const int h = key ? r - a.q.n : r - a.q.n - a.k.n;
    const Rows &in = key ? a.k : a.v;
    *p = {in.src + t * in.token + h * in.head, nullptr,
          (key ? a.cache.k : a.cache.v) + (int64_t)(slot >> a.cache.page_shift) * a.cache.page_stride +
              (int64_t)(slot & ((1 << a.cache.page_shift) - 1)) * a.cache.token_stride + h * a.cache.head_stride,
          key};
    return true;
}

// Any size and alignment: a wave per row.
template <int LAYOUT, bool BF16>
__global__ __launch_bounds__(THREADS) void rope_any_kernel(RopeArgs a) {
    const int64_t t = blockIdx.x;
    const int rows = a.q.n + a.k.n + a.v.n, wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const int slot = a.slots ? a.slots[t] : -1;
    for (int r = blockIdx.y * (THREADS / 64) + wave; r < rows; r += gridDim.y * (THREADS / 64)) {
        Place p;
        if (!place_of(a, t, r, slot, &p)) continue;
        if (p.to) row_any<LAYOUT, BF16>(a, p.from, p.to, a.pos[t], p.rotate, lane, 64);
        else row_any<LAYOUT, BF16>(a, p.from, p.stored, a.pos[t], p.rotate, lane, 64);
    }
}

// Eight elements of a row per thread, `units` threads a row, as many rows of
// one token at a time as fit; a thread's rows share its four turns.  Needs
// head_dim and n_dims multiples of 8 and 16-byte aligned rows.
template <int LAYOUT, bool BF16>
__global__ __launch_bounds__(THREADS) void rope_kernel(RopeArgs a, int units) {
    const int64_t t = blockIdx.x;
    const int unit = threadIdx.x % units, at_once = THREADS / units;
    if (threadIdx.x >= at_once * units) return;
    const int rows = a.q.n + a.k.n + a.v.n, slot = a.slots ? a.slots[t] : -1;
    const bool turned = unit < a.half / 4;  // else a unit behind the rotated elements
    const bool apart = LAYOUT == HIP_QMM_ROPE_HALF && turned;
    const int e0 = apart ? 4 * unit : 8 * unit, e1 = apart ? e0 + a.half : e0 + 4;  // the unit's two quads
    float c[4], s[4];
    if (turned) {
        const int64_t pos = a.pos[t];
#pragma unroll
        for (int i = 0; i < 4; ++i) turn(a, pos, 4 * unit + i, &c[i], &s[i]);
    }
    for (int r = threadIdx.x / units + at_once * blockIdx.y; r < rows; r += at_once * gridDim.y) {
        Place p;
        if (!place_of(a, t, r, slot, &p)) continue;
        const float4 x = *reinterpret_cast<const float4 *>(p.from + e0), y = *reinterpret_cast<const float4 *>(p.from + e1);
        float u[4] = {x.x, x.y, x.z, x.w}, v[4] = {y.x, y.y, y.z, y.w};
        if (turned && p.rotate) {
            float f[4], g[4];  // first and second members of the four pairs
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                f[j] = LAYOUT == HIP_QMM_ROPE_HALF ? u[j] : j < 2 ? u[2 * j] : v[2 * j - 4];
                g[j] = LAYOUT == HIP_QMM_ROPE_HALF ? v[j] : j < 2 ? u[2 * j + 1] : v[2 * j - 3];
            }
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float h = fmaf(f[j], c[j], -(g[j] * s[j]));
                g[j] = fmaf(f[j], s[j], g[j] * c[j]);
                f[j] = h;
            }
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                u[j] = LAYOUT == HIP_QMM_ROPE_HALF ? f[j] : j & 1 ? g[j >> 1] : f[j >> 1];
                v[j] = LAYOUT == HIP_QMM_ROPE_HALF ? g[j] : j & 1 ? g[2 + (j >> 1)] : f[2 + (j >> 1)];
            }
        }
        if (p.to) {
            *reinterpret_cast<float4 *>(p.to + e0) = make_float4(u[0], u[1], u[2], u[3]);
            *reinterpret_cast<float4 *>(p.to + e1) = make_float4(v[0], v[1], v[2], v[3]);
        } else {
            *reinterpret_cast<ushort4 *>(p.stored + e0) =
                make_ushort4(to16<BF16>(u[0]), to16<BF16>(u[1]), to16<BF16>(u[2]), to16<BF16>(u[3]));
            *reinterpret_cast<ushort4 *>(p.stored + e1) =
                make_ushort4(to16<BF16>(v[0]), to16<BF16>(v[1]), to16<BF16>(v[2]), to16<BF16>(v[3]));
        }
    }
}

bool aligned(const void *p, int64_t token, int64_t head) { return !((uintptr_t)p & 15) && !((token | head) & 3); }

template <int LAYOUT, bool BF16>
int launch(const RopeArgs &a, int64_t n_tokens, hipStream_t s) {
    const int rows = a.q.n + a.k.n + a.v.n;
    if (a.head_dim % 8 == 0 && a.half % 4 == 0 && aligned(a.q.src, a.q.token, a.q.head) &&
        aligned(a.dst, a.dst_token, a.dst_head) && aligned(a.k.src, a.k.token, a.k.head) && aligned(a.v.src, a.v.token, a.v.head)) {
        // A workgroup per token, or for few tokens one for each pass over its rows: of 8192, 1024 and 256 tokens'
        // 48 rows of 128 a workgroup per token took 69.1, 9.4 and 4.4 us, three per token 72.1, 11.0 and 4.3.
        const int units = a.head_dim / 8, at_once = THREADS / units;
        const int passes = n_tokens < FEW_TOKENS ? (rows + at_once - 1) / at_once : 1;
        hipLaunchKernelGGL((rope_kernel<LAYOUT, BF16>), dim3((unsigned)n_tokens, (unsigned)passes), dim3(THREADS), 0, s, a,
                           units);
    } else {
        const dim3 grid((unsigned)n_tokens, (unsigned)((rows + THREADS / 64 - 1) / (THREADS / 64)));
        hipLaunchKernelGGL((rope_any_kernel<LAYOUT, BF16>), grid, dim3(THREADS), 0, s, a);
    }
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
