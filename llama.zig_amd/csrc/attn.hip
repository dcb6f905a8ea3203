// attn.hip -- attention over the paged key-value cache: one pass over the keys
// and values of each sequence with the running maximum and sum of the softmax.
//
// The query rows of one key-value head are the (token, head) pairs of its
// group, token first: row r is token r / group, so that the heads of a group
// share every key and value that is read, for one token as for many.
//
// A wave contracts 16 rows or a few times as many with 32 tokens on 16x16x32
// matrix instructions, all transposed: scores S^T = K Q^T, results
// O^T = V^T P^T.  A row is then the lane index (mod 16) of both accumulators:
// maximum, sum and rescaling stay in the lane (but for one exchange among the
// four lane quarters that share a row), and the probabilities, as the scores
// lie, are the second operand of the next product: slot e of quarter g holds token
// 16*(e/4) + 4*g + e%4, an order that the transposing LDS reads of V follow.
//
// f32 results from 16-bit matrix cores: keys and values are what the cache
// holds, exactly; queries and probabilities go in as sums of PARTS 16-bit
// parts (two f16: 22 bits; three bf16: 24), each a product of its own into the
// f32 accumulators.  A query row is scaled by a power of two, and the
// probabilities carry another, so that the parts' range does not matter.
#include <math.h>

#include <algorithm>
#include <type_traits>

#include "kv_cache.h"

using namespace kvc;

namespace {

typedef float v2f __attribute__((ext_vector_type(2)));
typedef float v4f __attribute__((ext_vector_type(4)));
typedef uint32_t v2u __attribute__((ext_vector_type(2)));
typedef uint32_t v4u __attribute__((ext_vector_type(4)));
typedef _Float16 v2h __attribute__((ext_vector_type(2)));
typedef _Float16 v8h __attribute__((ext_vector_type(8)));
typedef __bf16 v2b __attribute__((ext_vector_type(2)));
typedef __bf16 v8b __attribute__((ext_vector_type(8)));
typedef short v4s __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) void *lds_ptr;
typedef __attribute__((address_space(3))) v4s *lds_v4s;

constexpr float LOG2E = 1.4426950408889634f;
constexpr float SLACK = 3.0f;   // the running maximum may lag by 2^SLACK

constexpr int MAX_LENGTH = 1 << 30;  // tokens of a sequence: sums of two positions fit 32 bits

struct AttnArgs {
    Cache c;
    const float *q;
    float *dst;
    int64_t q_token, q_head, dst_token, dst_head;
    const int32_t *q_starts, *table, *lens;
    int64_t table_stride;
    int n_seqs, n_heads, group, n_tokens;
    float scale;  // times log2(e)
    int window, sinks;
    int per, splits;       // tiles per split, splits at most
    int blocks;            // row blocks of a (sequence, key-value head)
    bool by_block;         // many rows: the last blocks of all pairs first, not pair after pair
    float *part_o, *part_ml;
};

// ---------------------------------------------------------------- 16-bit parts

template <bool BF16>
struct El;

template <>
struct El<false> {
    static constexpr int PARTS = 2;
    static constexpr uint32_t INF = 0x7c00;
    // A row of q is scaled to 2^QUERY and probabilities to 2^LIFT at the maximum: with SLACK both stay just below
    // f16's largest, and second parts and small weights lie as high above its smallest as they can.
    static constexpr int QUERY = 13;
    static constexpr float LIFT = 12.0f;
    static __device__ __forceinline__ v4f mma(v4u a, v4u b, v4f c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(v8h, a), __builtin_bit_cast(v8h, b), c, 0, 0, 0);
    }
    static __device__ __forceinline__ void split(float x, float y, uint32_t *p) {
        const v2h h = __builtin_convertvector((v2f){x, y}, v2h);
        p[0] = __builtin_bit_cast(uint32_t, h);
        v2f r;  // x - h.x, y - h.y, one mixed operation each
        asm("v_fma_mix_f32 %0, %1, -1.0, %2 op_sel:[0,0,0] op_sel_hi:[1,0,0]" : "=v"(r.x) : "v"(p[0]), "v"(x));
        asm("v_fma_mix_f32 %0, %1, -1.0, %2 op_sel:[1,0,0] op_sel_hi:[1,0,0]" : "=v"(r.y) : "v"(p[0]), "v"(y));
        p[1] = __builtin_bit_cast(uint32_t, __builtin_convertvector(r, v2h));
    }
};

template <>
struct El<true> {
    static constexpr int PARTS = 3;
    static constexpr uint32_t INF = 0x7f80;
    // Far below 1: sums over many of a cache's largest values (3e38) stay finite.
    static constexpr int QUERY = -10;
    static constexpr float LIFT = -16.0f;
    static __device__ __forceinline__ v4f mma(v4u a, v4u b, v4f c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(v8b, a), __builtin_bit_cast(v8b, b), c, 0, 0, 0);
    }
    static __device__ __forceinline__ void split(float x, float y, uint32_t *p) {
#pragma unroll
        for (int i = 0; i < 3; ++i) {
            p[i] = __builtin_bit_cast(uint32_t, __builtin_convertvector((v2f){x, y}, v2b));
            x -= __uint_as_float(p[i] << 16);
            y -= __uint_as_float(p[i] & 0xffff0000u);
        }
    }
};

// ---------------------------------------------------------------- what a block of rows sees

struct Seq {
    int first, m, n;  // its first row of q, its query count, its length
};

struct Rowspan {
    int first, m;
};

__device__ __forceinline__ Rowspan rows_of(const AttnArgs &a, int s) {
    if (!a.q_starts) return {s, 1};
    const int lo = max(a.q_starts[s], 0), hi = min(a.q_starts[s + 1], a.n_tokens);
    return {lo, max(hi - lo, 0)};
}

__device__ __forceinline__ Seq seq_of(const AttnArgs &a, const Rowspan &r, int s) {
    const int64_t most = min(a.table_stride << a.c.page_shift, (int64_t)MAX_LENGTH);
    return {r.first, r.m, (int)min((int64_t)max(a.lens[s], 0), most)};
}

__device__ __forceinline__ Seq seq_of(const AttnArgs &a, int s) { return seq_of(a, rows_of(a, s), s); }

// Rows [r0, r0 + rows) of a sequence's head group, their positions, and the
// tiles of TN tokens that any of them sees (from token `low` on, or one of the
// first): first `sink` tiles of the tokens that stay visible, then those from
// tile `from` on; `count` in all, dealt to the splits `per` at a time, `active`
// of which have some (the first always).
template <int TN>
struct Span {
    int rows, p_first, p_last, low, sink, from, count, per, active;

    __device__ __forceinline__ Span(const AttnArgs &a, const Seq &q, int r0, int block_rows) {
        rows = min(block_rows, q.m * a.group - r0);
        p_first = q.n - q.m + r0 / a.group;
        p_last = q.n - q.m + (r0 + rows - 1) / a.group;
        low = a.window ? max(0, p_first - a.window + 1) : 0;
        sink = (min(a.sinks, low) + TN - 1) / TN;
        from = max(low / TN, sink);
        count = p_last < 0 ? 0 : sink + max(0, p_last / TN + 1 - from);
        per = max(a.per, (count + a.splits - 1) / a.splits);
        active = max(1, (count + per - 1) / per);
    }
    __device__ __forceinline__ int token(int u) const { return (u < sink ? u : from + u - sink) * TN; }
};

// ---------------------------------------------------------------- LDS tiles

// A tile holds tokens as rows of DP elements in 16-byte chunks; chunk c of
// token t sits at c ^ swizzle(t), so that 16 tokens' reads of one chunk column
// meet all banks.
template <int DP>
__device__ __forceinline__ int swizzle(int t) { return DP == 64 ? (t >> 1) & 7 : t & 15; }

// 16 bytes per lane from base + off to LDS at lds_base + 16 * lane (base and
// lds_base wave-uniform).  Inline assembly, so that the compiler, which cannot
// tell the stages of a ring apart, puts no vmcnt(0) of its own before the LDS
// reads of another stage; every wait is wait_vm's.  M0 holds the LDS base.  The
// s_nop is what M0's write, and a base written by a vector instruction (lanes
// read back, as the compiler keeps scalars that do not fit), need before they
// are read, since it counts no wait states for an asm statement.
__device__ __forceinline__ void dma16(const uint16_t *base, uint32_t off, uint32_t lds_base) {
    asm volatile("s_nop 4\n\tglobal_load_lds_dwordx4 %0, %1" ::"v"(off), "s"(base), "{m0}"(lds_base) : "memory");
}

template <int N>
__device__ __forceinline__ void wait_vm() {
    static_assert(N >= 0 && N <= 63, "vmcnt field");
    __builtin_amdgcn_s_waitcnt(0x0F70 | (N & 15) | ((N >> 4) << 14));
    asm volatile("" ::: "memory");
}

__device__ __forceinline__ uint32_t lds_addr(const void *p) { return (uint32_t)(uintptr_t)(lds_ptr)p; }

// The page numbers of 64 consecutive entries of a sequence's table row, one
// per lane; an entry outside the pool or the row is -1.
struct Pages {
    const int32_t *row;
    int64_t width;
    int at, mine;

    __device__ __forceinline__ void load(int first, int n_pages) {
        at = first;
        const int i = at + (threadIdx.x & 63);
        const int e = i < width ? row[i] : -1;
        mine = (uint32_t)e < (uint32_t)n_pages ? e : -1;
    }
    // Entries i to i + more will be asked for (wave-uniform, more < 64).
    __device__ __forceinline__ void hold(int i, int more, int n_pages) {
        if (i < at || i + more > at + 63) load(i, n_pages);
    }
    __device__ __forceinline__ int get(int i) const { return __builtin_amdgcn_readlane(mine, i - at); }
};

// Transfers of 1024 bytes, PER tokens each, that fill tiles.  The lane's offset
// in a transfer depends on the transfer's number modulo NV alone: its chunk is
// its position XOR the token's swizzle, whose part from the lane and part from
// the transfer do not meet.  Chunks past the head repeat its last one.
template <int DP>
struct Loader {
    static constexpr int CH = DP / 8, PER = 64 / CH, NV = DP == 64 ? 2 : DP == 128 ? 4 : 8;
    static constexpr int GROUP = 16 / PER;  // transfers of 16 tokens, which are in one page
    uint32_t off[NV];

    __device__ __forceinline__ Loader(const AttnArgs &a) {
        const int lane = threadIdx.x & 63, t = lane / CH, last = (a.c.head_dim >> 3) - 1;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int chunk = min((lane % CH) ^ swizzle<DP>(i * PER + t), last);
            off[i] = ((uint32_t)t * (uint32_t)a.c.token_stride + chunk * 8) * 2;
        }
    }
    // 16 tokens from `base` to LDS.
    __device__ __forceinline__ void group(const AttnArgs &a, const uint16_t *base, uint32_t lds) const {
#pragma unroll
        for (int i = 0; i < GROUP; ++i) dma16(base + (int64_t)(i * PER) * a.c.token_stride, off[i % NV], lds + i * 1024);
    }
};

// Where tokens t0 to t0 + 15 of the held pages lie in a pool (a head's part added by the caller).
__device__ __forceinline__ int64_t group_at(const AttnArgs &a, int page, int t0) {
    return (int64_t)max(page, 0) * a.c.page_stride + (int64_t)(t0 & ((1 << a.c.page_shift) - 1)) * a.c.token_stride;
}

// ---------------------------------------------------------------- a wave's rows

// The larger of two, NaN if one is: unlike fmaxf it needs no operation that first quiets each matrix result.  (And no
// inline assembly on those: the compiler does not count it among the readers that wait for a matrix instruction.)
__device__ __forceinline__ float larger(float x, float y) { return __builtin_elementwise_maximum(x, y); }

// The largest of a value's four lane quarters, in all of them.
__device__ __forceinline__ float quarter_max(float m) {
    v2u x = __builtin_amdgcn_permlane16_swap(__float_as_uint(m), __float_as_uint(m), false, false);
    m = larger(__uint_as_float(x.x), __uint_as_float(x.y));
    x = __builtin_amdgcn_permlane32_swap(__float_as_uint(m), __float_as_uint(m), false, false);
    return larger(__uint_as_float(x.x), __uint_as_float(x.y));
}

// 16 * RT rows.  A tile's rows are DP = 64, 128 or 256 dimensions apart in LDS; DU of them, whole steps of a
// contraction, are worked on, and head_dim (DU, if FULL) are the head's.
template <bool BF16, int DP, int DU, bool FULL, int RT>
struct Rows {
    using E = El<BF16>;
    static constexpr int KS = DU / 32, DT = DU / 16, P = E::PARTS;

    v4u q[RT][P][KS];
    v4f o[RT][DT];
    float unit[RT];           // what a score is to be multiplied with: a power of two
    float top[RT], sum[RT];   // running maximum (log2), and this lane's share of the sum
    int pos[RT], low[RT];     // the row's position (-1: none), the first token of its window

    // Row 16 * i + lane % 16 of the block as it is, at x if it is valid.
    struct Raw {
        float v[KS][8];
    };
    static __device__ __forceinline__ Raw fetch(const AttnArgs &a, const float *x, bool valid) {
        const int g = (threadIdx.x & 63) >> 4, D = a.c.head_dim;
        Raw raw;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
            const int d = ks * 32 + g * 8;
            float4 u = make_float4(0.f, 0.f, 0.f, 0.f), w = u;
            if (valid && (FULL || d < D)) {
                u = *reinterpret_cast<const float4 *>(x + d);
                w = *reinterpret_cast<const float4 *>(x + d + 4);
            }
            float *v = raw.v[ks];
            v[0] = u.x, v[1] = u.y, v[2] = u.z, v[3] = u.w, v[4] = w.x, v[5] = w.y, v[6] = w.z, v[7] = w.w;
        }
        return raw;
    }

    // Its position (-1: none), its scale and its parts.
    __device__ __forceinline__ void take_row(const AttnArgs &a, int i, Raw &raw, int position) {
        auto &v = raw.v;
        float big = 0.0f;
        pos[i] = position;
        low[i] = a.window ? position - a.window + 1 : 0;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks)
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                v[ks][e] *= a.scale;
                big = fmaxf(big, fabsf(v[ks][e]));
            }
        big = quarter_max(big);
        const int ex = (int)(__float_as_uint(big) >> 23);  // biased; 255: not finite, left as it is
        // Not below -126, so that unit is finite: a largest query's parts then stay below 4.
        const int up = ex == 255 || ex == 0 ? 0 : max(min(E::QUERY - (ex - 127), 120), -126);
        unit[i] = ldexpf(1.0f, -up);
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
            uint32_t p[P];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                E::split(ldexpf(v[ks][2 * e], up), ldexpf(v[ks][2 * e + 1], up), p);
#pragma unroll
                for (int k = 0; k < P; ++k) q[i][k][ks][e] = p[k];
            }
        }
    }

    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int i = 0; i < RT; ++i) {
            top[i] = -INFINITY;
            sum[i] = 0.0f;
#pragma unroll
            for (int d = 0; d < DT; ++d) o[i][d] = (v4f){};
        }
    }

    // Scores of tokens [t, t + 32) of the tile: s[i][j] those of 16 j + 4 g + {0..3}.
    __device__ __forceinline__ void scores(const AttnArgs &a, const uint8_t *tile, int t, v4f (&s)[RT][2]) const {
        const int lane = threadIdx.x & 63, g = lane >> 4;
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const int tok = t + 16 * j + (lane & 15), sw = swizzle<DP>(tok);
            const uint8_t *row = tile + tok * (DP * 2);
#pragma unroll
            for (int i = 0; i < RT; ++i) s[i][j] = (v4f){};
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) {
                v4u k = *reinterpret_cast<const v4u *>(row + (((4 * ks + g) ^ sw) << 4));
                if (!FULL && ks * 32 + g * 8 >= a.c.head_dim) k = (v4u){};  // past the head: zeros, not its last chunk again
#pragma unroll
                for (int p = 0; p < P; ++p)
#pragma unroll
                    for (int i = 0; i < RT; ++i) s[i][j] = E::mma(k, q[i][p][ks], s[i][j]);
            }
        }
    }

    // The softmax's step over 32 tokens from t0 on: probabilities (times
    // 2^(LIFT - top)) in parts, the running values.
    __device__ __forceinline__ void soften(v4f (&s)[RT][2], v4u (&w)[RT][P]) {
        float m[RT];
        bool raise = false;
#pragma unroll
        for (int i = 0; i < RT; ++i) {
            float x = larger(s[i][0][0], s[i][0][1]);
#pragma unroll
            for (int r = 2; r < 8; ++r) x = larger(x, s[i][r >> 2][r & 3]);
            m[i] = quarter_max(x) * unit[i];  // NaN: not above top, and the row is NaN by its sum
            raise |= m[i] > top[i] + SLACK;
        }
        if (__any(raise)) {
#pragma unroll
            for (int i = 0; i < RT; ++i) {
                const bool mine = m[i] > top[i] + SLACK;
                const float shrink = mine ? __builtin_amdgcn_exp2f(top[i] - m[i]) : 1.0f;
                top[i] = mine ? m[i] : top[i];
                sum[i] *= shrink;
#pragma unroll
                for (int d = 0; d < DT; ++d) o[i][d] *= shrink;
            }
        }
#pragma unroll
        for (int i = 0; i < RT; ++i) {
            const float base = (top[i] == -INFINITY ? 0.0f : top[i]) - E::LIFT;
#pragma unroll
            for (int j = 0; j < 2; ++j) {
#pragma unroll
                for (int r = 0; r < 4; ++r) s[i][j][r] = __builtin_amdgcn_exp2f(fmaf(s[i][j][r], unit[i], -base));
                sum[i] += (s[i][j][0] + s[i][j][1]) + (s[i][j][2] + s[i][j][3]);
                uint32_t p[P];
#pragma unroll
                for (int r = 0; r < 4; r += 2) {
                    E::split(s[i][j][r], s[i][j][r + 1], p);
#pragma unroll
                    for (int k = 0; k < P; ++k) w[i][k][2 * j + (r >> 1)] = p[k];
                }
            }
        }
    }

    // The scores of tokens (t0 on) that their rows do not see; ok0, ok1: whether
    // the first and second 16 lie in the pool.
    __device__ __forceinline__ void hide(const AttnArgs &a, v4f (&s)[RT][2], int t0, bool ok0, bool ok1) const {
        const int g = (threadIdx.x & 63) >> 4;
#pragma unroll
        for (int i = 0; i < RT; ++i)
#pragma unroll
            for (int r = 0; r < 8; ++r) {
                const int t = t0 + 16 * (r >> 2) + 4 * g + (r & 3);
                const bool seen = (r < 4 ? ok0 : ok1) & (t <= pos[i]) & ((t >= low[i]) | (t < a.sinks));
                s[i][r >> 2][r & 3] = seen ? s[i][r >> 2][r & 3] : -INFINITY;
            }
    }

    // O^T += V^T P^T over tokens [t, t + 32) of the tile.
    __device__ __forceinline__ void gather(const uint8_t *tile, int t, const v4u (&w)[RT][P]) {
        const int lane = threadIdx.x & 63;
        const int ta = t + 4 * (lane >> 4) + ((lane & 15) >> 2), tb = ta + 16;
        const int sub = (lane & 3) >> 1;  // chunk inside 16 dimensions
        const uint8_t *ra = tile + ta * (DP * 2) + (lane & 1) * 8, *rb = ra + 16 * DP * 2;
        const int sa = swizzle<DP>(ta), sb = swizzle<DP>(tb);
        v4u v[DT];
#pragma unroll
        for (int d = 0; d < DT; ++d) {
            const v4s x = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s)(ra + (((2 * d + sub) ^ sa) << 4)));
            const v4s y = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s)(rb + (((2 * d + sub) ^ sb) << 4)));
            const v2u xu = __builtin_bit_cast(v2u, x), yu = __builtin_bit_cast(v2u, y);
            v[d] = (v4u){xu.x, xu.y, yu.x, yu.y};
        }
#pragma unroll
        for (int d = 0; d < DT; ++d)
#pragma unroll
            for (int p = 0; p < P; ++p)
#pragma unroll
                for (int i = 0; i < RT; ++i) o[i][d] = E::mma(v[d], w[i][p], o[i][d]);
    }

    // Whether some result is NaN: by a value that `Odd` would have kept apart, or rightly.
    __device__ __forceinline__ bool any_nan() const {
        bool nan = false;
#pragma unroll
        for (int i = 0; i < RT; ++i)
#pragma unroll
            for (int d = 0; d < DT; ++d)
#pragma unroll
                for (int r = 0; r < 4; ++r) nan |= o[i][d][r] != o[i][d][r];
        return __any(nan);
    }

    __device__ __forceinline__ float whole_sum(int i) const {
        const float x = sum[i] + __shfl_xor(sum[i], 16);
        return x + __shfl_xor(x, 32);
    }
};

// Whether some row of the span may not see some token of [t0, t0 + TN).
template <int TN>
__device__ __forceinline__ bool is_edge(const AttnArgs &a, const Span<TN> &sp, int t0) {
    return t0 + TN - 1 > sp.p_first || (a.window && t0 <= sp.p_last - a.window && t0 + TN > a.sinks);
}

// Row r of a sequence (a valid one): its query, and where its result goes.
__device__ __forceinline__ const float *query_row(const AttnArgs &a, const Seq &q, int kvh, int r) {
    const int t = r / a.group, g = r - t * a.group;
    return a.q + (int64_t)(q.first + t) * a.q_token + (int64_t)(kvh * a.group + g) * a.q_head;
}

__device__ __forceinline__ float *result_row(const AttnArgs &a, const Seq &q, int kvh, int r) {
    const int t = r / a.group, g = r - t * a.group;
    return a.dst + (int64_t)(q.first + t) * a.dst_token + (int64_t)(kvh * a.group + g) * a.dst_head;
}

__device__ __forceinline__ int64_t part_row(const AttnArgs &a, const Seq &q, int kvh, int r, int split) {
    const int t = r / a.group, g = r - t * a.group;
    return ((int64_t)split * a.n_tokens + q.first + t) * a.n_heads + kvh * a.group + g;
}

// Whether no row of the span sees some token of [t0, t0 + TN), `ok` aside.
template <int TN>
__device__ __forceinline__ bool has_unseen(const AttnArgs &a, const Span<TN> &sp, int t0) {
    return t0 + TN - 1 > sp.p_last || (t0 < sp.low && t0 + TN > a.sinks);
}

// Zeros for the values of tokens that no row sees, which may hold anything (their
// weight is 0, but 0 times infinity is not); by threads first, first + step, ...
template <int DP, int TN>
__device__ __forceinline__ void blank(const AttnArgs &a, const Span<TN> &sp, uint8_t *tile, int t0, int ok, int first,
                                      int step) {
    for (int i = first; i < TN * (DP / 8); i += step) {
        const int t = t0 + i / (DP / 8);
        if (!((ok >> ((t - t0) >> 4) & 1) && t <= sp.p_last && (t >= sp.low || t < a.sinks)))
            *reinterpret_cast<v4u *>(tile + i * 16) = (v4u){};
    }
}

// ---------------------------------------------------------------- keys and values that are not finite

// A value that some rows of a block see and others do not must not reach the
// others, where its weight is 0; and seen, it must not meet a weight's parts of
// both signs, nor an infinite key a query's parts.  No test for them is in the
// tiles' loops: a block whose results hold a NaN is done again, and then each
// tile's elements that are not finite become zeros before it is contracted, and
// are noted, in two bits each: inf and -inf, both for NaN and for a sum of the
// two.  Of values it is a row's and a dimension's, added to the results; of
// keys a row's and a token's, the query's element times the key's, added to the
// tile's scores; a NaN among a key's elements is the token's, whatever the row.
template <int DP, int ROWS, int TN>
struct Odd {
    static constexpr int WORDS = ROWS * DP / 16, NAN_KEYS = ROWS * TN / 16, KEY_WORDS = NAN_KEYS + TN / 32;
    uint32_t *bits, *key_bits;  // by row and dimension; by row and the tile's token, then a bit per token

    static __device__ __forceinline__ float number(uint32_t kind) {
        return kind == 1 ? INFINITY : kind == 2 ? -INFINITY : NAN;
    }

    // What is not finite in the tile of t0 becomes 0; note(row, token, dimension, kind) for each row that sees it, unless
    // done(token, whether it is NaN).  By threads first, first + step, ...; the block's rows begin at first_row of the
    // sequence, whose first position is p0.
    template <bool BF16, class Done, class Note>
    static __device__ __forceinline__ void sift(const AttnArgs &a, uint8_t *tile, int t0, int ok, int first_row, int rows,
                                                int first, int step, int p0, Done done, Note note) {
        constexpr uint32_t INF = El<BF16>::INF;
        for (int i = first; i < TN * (DP / 2); i += step) {
            uint32_t *w = reinterpret_cast<uint32_t *>(tile) + i;
            const uint32_t pair = *w;
            const bool lo = (pair & INF) == INF, hi = (pair >> 16 & INF) == INF;
            if (!lo && !hi) continue;
            *w = pair & (lo ? 0xffff0000u : ~0u) & (hi ? 0x0000ffffu : ~0u);
            const int t = i / (DP / 2), d = (((i & (DP / 2 - 1)) >> 2) ^ swizzle<DP>(t)) * 8 + (i & 3) * 2;
            if (!(ok >> (t >> 4) & 1) || d >= a.c.head_dim) continue;  // past the head: its last chunk again
            if (done(t, (pair & 0x7fffu) > INF || (pair >> 16 & 0x7fffu) > INF)) continue;
            for (int r = 0; r < rows; ++r) {
                const int p = p0 + (first_row + r) / a.group, j = t0 + t;
                if (!(j <= p && (!a.window || p - j < a.window || j < a.sinks))) continue;
                for (int e = 0; e < 2; ++e) {
                    const uint32_t b = pair >> (16 * e) & 0xffffu;
                    if ((b & INF) == INF) note(r, t, d + e, b == INF ? 1u : b == (INF | 0x8000u) ? 2u : 3u);
                }
            }
        }
    }
    __device__ __forceinline__ void clear_keys(int first, int step) const {
        for (int i = first; i < KEY_WORDS; i += step) key_bits[i] = 0;
    }
    // The tile's keys; rows of q from the sequence's on.
    template <bool BF16>
    __device__ __forceinline__ void sift_keys(const AttnArgs &a, const Seq &q, int kvh, uint8_t *tile, int t0, int ok,
                                              int first_row, int rows, int first, int step) const {
        auto done = [&](int t, bool nan) {
            uint32_t *w = &key_bits[NAN_KEYS + (t >> 5)];
            if (nan) atomicOr(w, 1u << (t & 31));
            return nan || (*w >> (t & 31) & 1);
        };
        sift<BF16>(a, tile, t0, ok, first_row, rows, first, step, q.n - q.m, done, [&](int r, int t, int d, uint32_t kind) {
            const float x = query_row(a, q, kvh, first_row + r)[d];
            if (x == 0.0f || x != x || a.scale == 0.0f) kind = 3;
            else if ((x < 0.0f) != (a.scale < 0.0f)) kind ^= 3;
            atomicOr(&key_bits[r * (TN / 16) + (t >> 4)], kind << (2 * (t & 15)));
        });
    }
    // The tile's values, after its keys: times a weight of exactly 0 (a score of -inf) an infinity is NaN.
    template <bool BF16>
    __device__ __forceinline__ void sift_values(const AttnArgs &a, const Seq &q, uint8_t *tile, int t0, int ok,
                                                int first_row, int rows, int first, int step) const {
        auto done = [](int, bool) { return false; };
        sift<BF16>(a, tile, t0, ok, first_row, rows, first, step, q.n - q.m, done, [&](int r, int t, int d, uint32_t kind) {
            if (key_bits[r * (TN / 16) + (t >> 4)] >> (2 * (t & 15)) & 3) kind = 3;
            atomicOr(&bits[r * (DP / 16) + (d >> 4)], kind << (2 * (d & 15)));
        });
    }
    // Scores of the tile's tokens [t, t + 32), as Rows::scores leaves them, for rows from r0 on.
    template <int RT>
    __device__ __forceinline__ void apply_keys(int r0, int t, v4f (&s)[RT][2]) const {
        int lane = threadIdx.x & 63;
        asm("" : "+v"(lane));  // nothing of this is computed ahead of the tiles' loop, whose registers are full
#pragma unroll
        for (int i = 0; i < RT; ++i)
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const uint32_t k = key_bits[(r0 + 16 * i + (lane & 15)) * (TN / 16) + (t >> 4) + j] >> (8 * (lane >> 4));
                const uint32_t nan = key_bits[NAN_KEYS + (t >> 5)] >> (16 * j + 4 * (lane >> 4));
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    if (k >> (2 * e) & 3) s[i][j][e] += number(k >> (2 * e) & 3);
                    if (nan >> e & 1) s[i][j][e] = NAN;
                }
            }
    }
    // Row r's dimension d, given its result without them.
    __device__ __forceinline__ float apply(int r, int d, float x) const {
        const uint32_t k = bits[r * (DP / 16) + (d >> 4)] >> (2 * (d & 15)) & 3;
        return k == 0 ? x : x + number(k);
    }
};

// What results under the maximum `top` count for under `m`: never 0, which would make a NaN of one that is infinite,
// however small its share.
__device__ __forceinline__ float weight_of(float top, float m) {
    return fmaxf(__builtin_amdgcn_exp2f(top - m), 0x1p-126f);
}

// ---------------------------------------------------------------- few rows

// 16 * RT rows (one token's heads, or a few tokens'): bound by the reads of K
// and V, and where those are few by the chain of dependent loads (length, page
// numbers, keys).  Every wave has tiles of 32 tokens of its own, in a ring of
// ST stages whose K and V halves are refilled as soon as they have been read,
// with no barrier.  At the end the waves' results are joined in LDS.
//
// 32 query heads on 8 of 128 dimensions, f16: 131072 tokens (537 MB) 98 us, 5.5
// TB/s (a large copy: 5.3); 16384 18.6; 4096 11.8; 333 8.7, where a launch is
// 2.5.  100 sequences of a 1024-token window with 32 heads of 64 (819 MB): 148
// us, 5.5 TB/s.  48 of up to 8191 in bf16 (447 MB): 97 us, 4.6 TB/s, with the
// join's 5 us.  Four waves with one stage leave room for two workgroups a CU:
// two stages took 9.4, 11.8 and 108 us for 333 tokens, 4096 and the 48, eight
// waves 8.0, 12.0 and 105.  With many short sequences NW is 1 (`plan_of`).
template <int DP, int RT, int NW>
struct Few {
    static constexpr int TN = 32, ST = DP == 64 ? 2 : 1, HALF = TN * DP * 2;
    static constexpr int NX = HALF / 1024;     // transfers per half
    static constexpr int OS = DP + 4;          // floats of a row of results, off the banks' period
    static constexpr int RING = 2 * ST * HALF > 16 * RT * OS * 4 ? 2 * ST * HALF : 16 * RT * OS * 4;
};

template <bool BF16, int DP, int DU, bool FULL, int RT, int NW>
__global__ __launch_bounds__(64 * NW, RT * DP <= 128 ? 2 : 1) void few_kernel(AttnArgs a) {
    using F = Few<DP, RT, NW>;
    __shared__ __attribute__((aligned(1024))) uint8_t ring[NW][F::RING];
    __shared__ float tops[NW][16 * RT], sums[NW][16 * RT];
    using O = Odd<DP, 16 * RT, F::TN>;
    __shared__ uint32_t odd_bits[O::WORDS], odd_keys[NW][O::KEY_WORDS];
    // Workgroups are dealt to the eight XCDs in turn, and the later splits of short sequences are empty: splits
    // slowest (first, four of them, XCDs 3 and 7 had only the longest sequences' last quarters), and where that would
    // leave all splits of a sequence to the same few XCDs each split begins with another sequence (48 of up to 8191
    // tokens, 4 heads: 100.7 -> 97.8 us).
    const int per_seq = a.c.n_kv_heads * a.blocks, pairs = a.n_seqs * per_seq;
    const int split = blockIdx.x / pairs, pair = blockIdx.x - split * pairs, turn = pair / per_seq;
    const int seq = (pairs & 7) == 0 && (per_seq & 7) ? (turn + split) % a.n_seqs : turn;
    const int kvh = (pair - turn * per_seq) / a.blocks, block = pair - turn * per_seq - kvh * a.blocks;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    const int r0 = block * (16 * RT);
    const O odd = {odd_bits, odd_keys[wave]};
    // Three loads that do not wait for one another: the rows, the length, and
    // the pages of the tile that is this wave's first where the length does
    // not change the split and there is no window.
    const Rowspan own = rows_of(a, seq);
    if (r0 >= own.m * a.group) return;
    typename Rows<BF16, DP, DU, FULL, RT>::Raw raw[RT];
#pragma unroll
    for (int i = 0; i < RT; ++i) {
        const int row = r0 + 16 * i + (lane & 15), tok = row / a.group;
        raw[i] = Rows<BF16, DP, DU, FULL, RT>::fetch(
            a, a.q + (int64_t)(own.first + tok) * a.q_token + (int64_t)(kvh * a.group + row - tok * a.group) * a.q_head,
            row < own.m * a.group);
    }
    Pages pages = {a.table + seq * a.table_stride, a.table_stride, 0, -1};
    pages.load((split * a.per + wave) * F::TN >> a.c.page_shift, a.c.n_pages);
    const Seq q = seq_of(a, own, seq);
    const Span<F::TN> sp(a, q, r0, 16 * RT);
    if (split >= sp.active) return;

    const int64_t head = (int64_t)kvh * a.c.head_stride;
    const int begin = split * sp.per + wave, end = min(sp.count, (split + 1) * sp.per);
    const int tiles = begin < end ? (end - begin + NW - 1) / NW : 0;
    const uint32_t lds = __builtin_amdgcn_readfirstlane(lds_addr(ring[wave]));
    const Loader<DP> loader(a);
    const int more = a.c.page_shift == 4 ? 1 : 0;  // a tile spans two pages of 16 tokens
    uint32_t oks = 0;  // two bits per stage
    int64_t at0 = 0, at1 = 0;  // where the tile last begun lies

    auto issue_keys = [&](int i) {
        const int t0 = sp.token(begin + i * NW), p = t0 >> a.c.page_shift, st = i % F::ST;
        pages.hold(p, more, a.c.n_pages);
        const int p0 = pages.get(p), p1 = pages.get(p + more);
        const uint32_t ok = (p0 >= 0 ? 1 : 0) | (p1 >= 0 ? 2 : 0);
        oks = (oks & ~(3u << (2 * st))) | ok << (2 * st);
        at0 = head + group_at(a, p0, t0);
        at1 = head + group_at(a, p1, t0 + 16);
        loader.group(a, a.c.k + at0, lds + st * 2 * F::HALF);
        loader.group(a, a.c.k + at1, lds + st * 2 * F::HALF + F::HALF / 2);
    };
    auto issue_values = [&](int i) {  // of the tile that issue_keys last began
        const int st = i % F::ST;
        loader.group(a, a.c.v + at0, lds + (st * 2 + 1) * F::HALF);
        loader.group(a, a.c.v + at1, lds + (st * 2 + 1) * F::HALF + F::HALF / 2);
    };
    // At most n halves issued after the one wanted may be outstanding.
    auto wait_halves = [&](int n) {
        if (F::ST > 1 && n >= 3) wait_vm<3 * F::NX>();
        else if (F::ST > 1 && n == 2) wait_vm<2 * F::NX>();
        else if (n >= 1) wait_vm<F::NX>();
        else wait_vm<0>();
    };
    auto start = [&] {
#pragma unroll
        for (int i = 0; i < F::ST; ++i)
            if (i < tiles) {
                issue_keys(i);
                issue_values(i);
            }
    };
    Rows<BF16, DP, DU, FULL, RT> w;
#pragma unroll
    for (int i = 0; i < RT; ++i) {
        const int in = 16 * i + (lane & 15);
        w.take_row(a, i, raw[i], in < sp.rows ? q.n - q.m + (r0 + in) / a.group : -1);
    }
    // One pass over the tiles, and the join of the waves; whether some result is NaN.  Two copies of the code: the first
    // pass keeps the registers of a loop that cares for nothing.
    auto pass = [&](auto careful) {
        constexpr bool care = decltype(careful)::value;
        w.clear();
        if (tiles > 0) start();
        for (int i = 0; i < tiles; ++i) {
            const int t0 = sp.token(begin + i * NW), st = i % F::ST;
            const bool ok0 = oks >> (2 * st) & 1, ok1 = oks >> (2 * st) & 2;
            uint8_t *k = ring[wave] + st * 2 * F::HALF, *v = k + F::HALF;
            const int after = 2 * (tiles - i) - 1;  // halves to come after this tile's keys, those not yet issued too
            wait_halves(min(after, 2 * F::ST - 1));
            v4f s[RT][2];
            v4u p[RT][El<BF16>::PARTS];
            if (care) {
                odd.clear_keys(lane, 64);
                asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
                odd.template sift_keys<BF16>(a, q, kvh, k, t0, ok0 | ok1 << 1, r0, sp.rows, lane, 64);
                asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
            }
            w.scores(a, k, 0, s);
            if (care) odd.apply_keys(0, 0, s);
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // the keys have been read: their half may be refilled
            if (i + F::ST < tiles) issue_keys(i + F::ST);
            if (is_edge<F::TN>(a, sp, t0) || !(ok0 && ok1)) w.hide(a, s, t0, ok0, ok1);
            w.soften(s, p);
            wait_halves(min(after - 1, 2 * F::ST - 1));
            if (care || has_unseen<F::TN>(a, sp, t0) || !(ok0 && ok1)) {
                blank<DP, F::TN>(a, sp, v, t0, ok0 | ok1 << 1, lane, 64);
                if (care) odd.template sift_values<BF16>(a, q, v, t0, ok0 | ok1 << 1, r0, sp.rows, lane, 64);
                asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
            }
            w.gather(v, 0, p);
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
            if (i + F::ST < tiles) issue_values(i + F::ST);
        }

        // Join the waves: every one's O in its own ring (its transfers are done).
        float *mine = reinterpret_cast<float *>(ring[wave]);
#pragma unroll
        for (int i = 0; i < RT; ++i) {
            const int in = 16 * i + (lane & 15);
            const float l = w.whole_sum(i);
            if (lane < 16) {
                tops[wave][in] = w.top[i];
                sums[wave][in] = l;
            }
            if (in < sp.rows) {
#pragma unroll
                for (int d = 0; d < DU / 16; ++d)
                    *reinterpret_cast<v4f *>(mine + in * F::OS + d * 16 + 4 * (lane >> 4)) = w.o[i][d];
            }
        }
        __syncthreads();
        const int quads = a.c.head_dim >> 2;
        bool nan = false;
        for (int i = threadIdx.x; i < sp.rows * quads; i += NW * 64) {
            const int r = i / quads, d = (i - r * quads) * 4;
            float m = -INFINITY;
#pragma unroll
            for (int k = 0; k < NW; ++k) m = fmaxf(m, tops[k][r]);
            v4f o = {};
            float total = 0.0f;
#pragma unroll
            for (int k = 0; k < NW; ++k) {
                if (tops[k][r] == -INFINITY && sums[k][r] == 0.0f) continue;  // nothing seen
                const float f = __builtin_amdgcn_exp2f(tops[k][r] - m);
                const v4f u = *reinterpret_cast<const v4f *>(reinterpret_cast<const float *>(ring[k]) + r * F::OS + d);
                total = fmaf(f, sums[k][r], total);
                o += f * u;
            }
            if (care) {
#pragma unroll
                for (int e = 0; e < 4; ++e) o[e] = odd.apply(r, d + e, o[e]);
            }
            nan |= o[0] != o[0] || o[1] != o[1] || o[2] != o[2] || o[3] != o[3];
            if (sp.active == 1) {
                o = total == 0.0f ? (v4f){} : o / total;
                *reinterpret_cast<v4f *>(result_row(a, q, kvh, r0 + r) + d) = o;
            } else {
                const int64_t at = part_row(a, q, kvh, r0 + r, split);
                *reinterpret_cast<v4f *>(a.part_o + at * a.c.head_dim + d) = o;
                if (d == 0) *reinterpret_cast<float2 *>(a.part_ml + at * 2) = make_float2(m, total);
            }
        }
        return nan;
    };
    if (!__syncthreads_or(pass(std::false_type{}))) [[likely]] return;
    for (int i = threadIdx.x; i < O::WORDS; i += NW * 64) odd_bits[i] = 0;
    __syncthreads();
    pass(std::true_type{});
}

// ---------------------------------------------------------------- many rows

// 128 rows, 32 per wave, against tiles of 64 tokens that the four waves share:
// bound by the matrix cores and the softmax beside them, whose times add up on
// this part (a prompt of 4096 tokens, 32 heads on 8 of 128 in f16: 258 us, 533
// TFLOP/s of the one product that counts, 1066 of the two that run; matrix
// instructions are 45 % of the cycles, vector ones 31).  A row takes 5 to 6
// vector operations per score, of which the exponential counts for four, so
// that 16 rows a wave, which would double the reads of LDS, or parts of P
// passed through LDS gain nothing.
// Two stages: the next tile's transfers are in flight while one is contracted,
// one barrier per tile.  With 64 rows two waves have the same rows and half of
// the tokens each, and are joined at the end (WT = 2).  For 256 dimensions only
// 64 rows, 16 per wave, and tiles of 32 tokens: two workgroups fit a CU, in 256
// registers a lane, none in memory.  (With 32 rows per wave and tiles of 64 one
// did: 2048 tokens 183 us in f16 and 360 in bf16, not 151 and 177; 13 tokens on
// 20000 102 and 265, not 67 and 75.)
template <int DP, int ROWS>
struct Many {
    static constexpr bool WIDE = DP == 256;
    static constexpr int TN = WIDE ? 32 : 64, NW = 4, RT = WIDE ? 1 : 2, WT = NW * 16 * RT / ROWS;
    static constexpr int GROUPS = TN / 16, ALL = (1 << GROUPS) - 1, HALF = TN * DP * 2, STAGE = 2 * HALF;
};

template <bool BF16, int DP, int DU, bool FULL, int ROWS>
__global__ __launch_bounds__(256, 2) void many_kernel(AttnArgs a) {
    using M = Many<DP, ROWS>;
    constexpr int WT = M::WT;
    __shared__ __attribute__((aligned(1024))) uint8_t stage[2][M::STAGE];
    using O = Odd<DP, ROWS, M::TN>;
    __shared__ uint32_t odd_bits[O::WORDS], odd_keys[O::KEY_WORDS];
    const O odd = {odd_bits, odd_keys};
    const int split = blockIdx.y;
    // Workgroups are dealt to the eight XCDs in turn.  Blocks of one key-value head share its keys and values, so a
    // head goes to one XCD, or to 8 / n of them in turn; and every sequence to all of them, as its length may be any
    // (three windowed prompts of up to 2500 tokens, 4 heads: 178 us, 217 with each pair of both on one XCD; eight of
    // up to 1000 with one head 97 and 153).
    const int H = a.c.n_kv_heads, n = min(H & -H, 8), xcd = blockIdx.x & 7;
    const int id = (blockIdx.x >> 3) * (8 / n) + xcd / n, pairs = H / n * a.n_seqs;
    const int block = a.by_block ? id / pairs : id % a.blocks;
    const int pair = a.by_block ? (id + block) % pairs : id / a.blocks;
    const int s = pair / (H / n), kvh = (pair - s * (H / n)) * n + xcd % n;
    const Seq q = seq_of(a, s);
    const int all = q.m * a.group, mine = (all + ROWS - 1) / ROWS;
    if (block >= mine) return;
    const int r0 = (mine - 1 - block) * ROWS;  // the last rows see most: first
    const Span<M::TN> sp(a, q, r0, ROWS);
    if (split >= sp.active) return;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;

    const int64_t head = (int64_t)kvh * a.c.head_stride;
    const int begin = split * sp.per, end = min(sp.count, begin + sp.per);
    Pages pages = {a.table + s * a.table_stride, a.table_stride, 0, -1};
    const Loader<DP> loader(a);
    const int more = max((M::TN >> a.c.page_shift) - 1, 0);
    uint32_t oks = 0;  // GROUPS bits per stage
    // Wave w transfers tokens 16 w to 16 w + 15, of two groups either the keys or the values.
    auto issue = [&](int u) {
        const int t0 = sp.token(u), p = t0 >> a.c.page_shift;
        pages.hold(p, more, a.c.n_pages);
        uint32_t ok = 0;
#pragma unroll
        for (int g = 0; g < M::GROUPS; ++g) ok |= pages.get((t0 + 16 * g) >> a.c.page_shift) >= 0 ? 1u << g : 0;
        oks = u & 1 ? (oks & M::ALL) | ok << M::GROUPS : (oks & M::ALL << M::GROUPS) | ok;
        const int g = wave % M::GROUPS, t = t0 + 16 * g;
        const uint32_t lds = __builtin_amdgcn_readfirstlane(lds_addr(stage[u & 1])) + g * (M::HALF / M::GROUPS);
        const int64_t at = head + group_at(a, pages.get(t >> a.c.page_shift), t);
        if constexpr (M::GROUPS == M::NW) {
            loader.group(a, a.c.k + at, lds);
            loader.group(a, a.c.v + at, lds + M::HALF);
        } else if (wave < M::GROUPS) {
            loader.group(a, a.c.k + at, lds);
        } else {
            loader.group(a, a.c.v + at, lds + M::HALF);
        }
    };
    auto start = [&] {
        pages.load(sp.token(begin) >> a.c.page_shift, a.c.n_pages);
        issue(begin);
    };
    if (begin < end) start();
    Rows<BF16, DP, DU, FULL, M::RT> w;
#pragma unroll
    for (int i = 0; i < M::RT; ++i) {
        const int in = wave % (M::NW / WT) * (16 * M::RT) + 16 * i + (lane & 15), row = r0 + in, tok = row / a.group;
        auto raw = w.fetch(
            a, a.q + (int64_t)(q.first + tok) * a.q_token + (int64_t)(kvh * a.group + row - tok * a.group) * a.q_head,
            in < sp.rows);
        w.take_row(a, i, raw, in < sp.rows ? q.n - q.m + tok : -1);
    }
    // One pass over the tiles.  Two copies of the code: the first pass keeps the registers of a loop that cares for nothing.
    auto pass = [&](auto careful) {
        constexpr bool care = decltype(careful)::value;
        w.clear();
        for (int u = begin; u < end; ++u) {
            wait_vm<0>();
            __builtin_amdgcn_s_waitcnt(0xC07F);  // lgkmcnt(0): this wave has read the stage that is refilled next
            __builtin_amdgcn_s_barrier();
            asm volatile("" ::: "memory");
            const int ok = oks >> (M::GROUPS * (u & 1)) & M::ALL, t0 = sp.token(u);
            if (u + 1 < end) issue(u + 1);
            uint8_t *k = stage[u & 1], *v = k + M::HALF;
            if (care) {
                odd.clear_keys(threadIdx.x, 256);
                __syncthreads();
                odd.template sift_keys<BF16>(a, q, kvh, k, t0, ok, r0, sp.rows, threadIdx.x, 256);
                __syncthreads();
            }
            if (care || has_unseen<M::TN>(a, sp, t0) || ok != M::ALL) {
                blank<DP, M::TN>(a, sp, v, t0, ok, threadIdx.x, 256);
                if (care) odd.template sift_values<BF16>(a, q, v, t0, ok, r0, sp.rows, threadIdx.x, 256);
                asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
            }
            const bool edge = is_edge<M::TN>(a, sp, t0) || ok != M::ALL;
            auto half = [&](int i) {
                v4f x[M::RT][2];
                v4u p[M::RT][El<BF16>::PARTS];
                w.scores(a, k, 32 * i, x);
                if (care) odd.apply_keys(wave % (M::NW / WT) * (16 * M::RT), 32 * i, x);
                if (edge) w.hide(a, x, t0 + 32 * i, ok >> (2 * i) & 1, ok >> (2 * i + 1) & 1);
                // Matrix instructions first where the SIMD's other wave is at its softmax (274 -> 267 us for a
                // prompt of 4096 tokens in f16, 353 -> 340 in bf16).
                __builtin_amdgcn_s_setprio(0);
                w.soften(x, p);
                __builtin_amdgcn_s_setprio(1);
                w.gather(v, 32 * i, p);
            };
            if constexpr (WT == 2) {
                half(wave >> 1);
            } else {
#pragma unroll 1
                for (int i = 0; i < M::TN / 32; ++i) half(i);
            }
        }
    };
    pass(std::false_type{});
    const bool care = __syncthreads_or(w.any_nan());
    if (care) [[unlikely]] {
        for (int i = threadIdx.x; i < O::WORDS; i += 256) odd_bits[i] = 0;
        __syncthreads();  // (which also frees both stages)
        if (begin < end) start();
        pass(std::true_type{});
        __syncthreads();  // as after the first pass: the join below writes over the stages
    }
    if constexpr (WT == 2) {  // the stages are free: each pass ended in a barrier
        v4f *other = reinterpret_cast<v4f *>(stage[0]) + (wave & 1) * 64 * M::RT * (DU / 16 + 1) + lane;
        if (wave >= 2) {
#pragma unroll
            for (int i = 0; i < M::RT; ++i) {
#pragma unroll
                for (int d = 0; d < DU / 16; ++d) other[(i * (DU / 16 + 1) + d) * 64] = w.o[i][d];
                other[(i * (DU / 16 + 1) + DU / 16) * 64] = (v4f){w.top[i], w.sum[i], 0.0f, 0.0f};
            }
        }
        __syncthreads();
        if (wave >= 2) return;
#pragma unroll
        for (int i = 0; i < M::RT; ++i) {
            const v4f ts = other[(i * (DU / 16 + 1) + DU / 16) * 64];
            // A lane's share of a sum is 0 where its row saw nothing; the others' of the row then too.
            const float top = fmaxf(w.top[i], ts[0]), base = top == -INFINITY ? 0.0f : top;
            const float f = weight_of(w.top[i], base), g = weight_of(ts[0], base);
            w.sum[i] = f * w.sum[i] + g * ts[1];
            w.top[i] = top;
#pragma unroll
            for (int d = 0; d < DU / 16; ++d) w.o[i][d] = f * w.o[i][d] + g * other[(i * (DU / 16 + 1) + d) * 64];
        }
    }

#pragma unroll
    for (int i = 0; i < M::RT; ++i) {
        const int in = wave % (M::NW / WT) * (16 * M::RT) + 16 * i + (lane & 15), row = r0 + in;
        const float total = w.whole_sum(i);
        if (in >= sp.rows) continue;
        float *out;
        float f = 1.0f;
        if (sp.active == 1) {
            out = result_row(a, q, kvh, row);
            f = total == 0.0f ? 0.0f : 1.0f / total;
        } else {
            const int64_t at = part_row(a, q, kvh, row, split);
            out = a.part_o + at * a.c.head_dim;
            if (lane < 16) *reinterpret_cast<float2 *>(a.part_ml + at * 2) = make_float2(w.top[i], total);
        }
#pragma unroll
        for (int d = 0; d < DU / 16; ++d) {
            const int e = d * 16 + 4 * (lane >> 4);
            v4f x = w.o[i][d] * f;
            if (care && (sp.active > 1 || total != 0.0f)) {
#pragma unroll
                for (int c = 0; c < 4; ++c) x[c] = odd.apply(in, e + c, x[c]);
            }
            if (FULL || e < a.c.head_dim) *reinterpret_cast<v4f *>(out + e) = x;
        }
    }
}

// ---------------------------------------------------------------- join of the splits

// A launch of its own: bound by its latency, 4 to 6 us.  (Joined in the same
// launch by the last workgroup of a row, the flags' release and acquire wrote
// the XCDs' L2 back and took longer: 16384 tokens 73 us instead of 19.)
// For many splits one workgroup per row.  The weights of the splits first (in
// LDS), then their results: LANES threads hold a row, the groups of them take
// the splits in turn, four loads of each in flight, and are added in order.
constexpr int MAX_SPLITS = 256, SOME_SPLITS = 16;

__device__ __forceinline__ float split_weight(float2 p, float m) {
    return p.x == -INFINITY && p.y == 0.0f ? 0.0f : weight_of(p.x, m);  // a split that saw nothing: 0, and zeros
}

template <int TN, int ROWS, int LANES>
__global__ __launch_bounds__(256) void join_kernel(AttnArgs a) {
    __shared__ float weight[MAX_SPLITS], part[8];
    __shared__ v4f sums[256];
    const Seq q = seq_of(a, blockIdx.z);
    const int kvh = blockIdx.y, r = blockIdx.x, tid = threadIdx.x, wave = tid >> 6;
    if (r >= q.m * a.group) return;
    const Span<TN> sp(a, q, r / ROWS * ROWS, ROWS);
    if (sp.active == 1) return;
    const int64_t step = (int64_t)a.n_tokens * a.n_heads, at = part_row(a, q, kvh, r, 0);
    const float2 p = tid < sp.active ? reinterpret_cast<const float2 *>(a.part_ml)[at + tid * step]
                                     : make_float2(-INFINITY, 0.0f);
    float m = p.x;
    for (int o = 32; o; o >>= 1) m = fmaxf(m, __shfl_xor(m, o));
    if ((tid & 63) == 0) part[wave] = m;
    __syncthreads();
    m = fmaxf(fmaxf(part[0], part[1]), fmaxf(part[2], part[3]));
    const float f = split_weight(p, m);
    float total = f == 0.0f ? 0.0f : f * p.y;
    weight[tid] = f;
    for (int o = 32; o; o >>= 1) total += __shfl_xor(total, o);
    if ((tid & 63) == 0) part[4 + wave] = total;
    __syncthreads();
    constexpr int GROUPS = 256 / LANES;
    const int D = a.c.head_dim, d = tid % LANES * 4;
    v4f o = {};
    if (d < D) {
        const float *src = a.part_o + at * D + d;
#pragma unroll 4
        for (int k = tid / LANES; k < sp.active; k += GROUPS) o += weight[k] * *reinterpret_cast<const v4f *>(src + k * step * D);
    }
    sums[tid] = o;
    __syncthreads();
    if (tid >= LANES || d >= D) return;
    total = (part[4] + part[5]) + (part[6] + part[7]);
#pragma unroll
    for (int k = 1; k < GROUPS; ++k) o += sums[k * LANES + tid];
    *reinterpret_cast<v4f *>(result_row(a, q, kvh, r) + d) = total == 0.0f ? (v4f){} : o / total;
}

// For at most SOME_SPLITS of them LANES threads per row and nothing shared (48 sequences of 4 splits: 5.0 us).
template <int TN, int ROWS, int LANES>
__global__ __launch_bounds__(256) void join_some_kernel(AttnArgs a) {
    const Seq q = seq_of(a, blockIdx.z);
    const int kvh = blockIdx.y, r = blockIdx.x * (256 / LANES) + threadIdx.x / LANES, d = threadIdx.x % LANES * 4;
    if (r >= q.m * a.group) return;
    const Span<TN> sp(a, q, r / ROWS * ROWS, ROWS);
    const int D = a.c.head_dim;
    if (sp.active == 1 || d >= D) return;
    const int64_t step = (int64_t)a.n_tokens * a.n_heads, at = part_row(a, q, kvh, r, 0);
    const float2 *ml = reinterpret_cast<const float2 *>(a.part_ml) + at;
    float m = -INFINITY;
#pragma unroll 4
    for (int k = 0; k < sp.active; ++k) m = fmaxf(m, ml[k * step].x);
    const float *src = a.part_o + at * D + d;
    v4f o = {};
    float total = 0.0f;
#pragma unroll 4
    for (int k = 0; k < sp.active; ++k) {
        const float2 p = ml[k * step];
        const v4f u = *reinterpret_cast<const v4f *>(src + k * step * D);
        const float f = split_weight(p, m);
        total = fmaf(f, p.y, total);
        o += f * u;
    }
    *reinterpret_cast<v4f *>(result_row(a, q, kvh, r) + d) = total == 0.0f ? (v4f){} : o / total;
}

// ---------------------------------------------------------------- host

struct Plan {
    int rows;  // of a block: 16 or 32 (few), 64 or 128; 16 or 64 for over 128 dimensions
    int blocks, per, splits;
    int waves;  // of a few-row workgroup: 1 or 4
    bool by_block;
    bool few() const { return rows <= 32; }
};

// Tiles per split of the few-row kernel.  A workgroup per CU reads as fast as
// two do, and a split's cost is its start and the join: 8 heads of 131072 tokens
// in splits of 16, 32, 64, 128, 256 and 512 tiles took 110, 106, 101, 99, 104
// and 174 us, of 4096 tokens in 4, 8, 16, 32 and 64 13.1, 13.5, 15.3, 20.2 and
// 30.0.  Sequences of unlike lengths leave some workgroups little, so no more
// than 64 tiles where there are several: 48 of up to 8191 in 32, 64, 192 and 256
// took 105, 104, 110 and 109 us.  Up to 14 tiles the join costs more than it
// saves: 333 tokens in 4, 8 and all at once 11.4, 12.0 and 10.5 us.
int64_t few_per(int64_t tiles, int64_t grid, int64_t n_seqs) {
    if (tiles <= 14) return tiles;
    const int64_t per = ((tiles * grid + 255) / 256 + 3) / 4 * 4;
    return n_seqs > 1 && per > 64 ? 64 : per;
}

// Of the many-row kernel with 128 rows, and the time in us: a tile takes 2.9
// alone on a CU, 4.2 beside another workgroup, and splits their results, written
// and read once, and the join.  512 workgroups are two a CU; the share is exact
// rather than a power of two.
int64_t many_per(int64_t tiles, int64_t grid, double result_bytes, double *time) {
    int64_t per = tiles;
    double best = (grid <= 256 ? 2.9 : 4.2) * (double)tiles;
    for (int64_t n = 2; n * grid <= 512 && n <= MAX_SPLITS; n *= 2) {
        const int64_t each = (tiles + n - 1) / n;
        const double t = 2.9 * (double)each + 8.0 + result_bytes * (double)n / 4e6;
        if (each < 2 || t >= best) continue;
        best = t;
        per = each;
    }
    *time = best;
    return per < tiles ? std::max((tiles * grid + 511) / 512, std::min(per, (int64_t)2)) : tiles;
}

constexpr int64_t MAX_GROUPS = 1 << 23;  // workgroups of a launch

// Which kernel, its rows per workgroup, and how the tokens are split; rows is 0 where even unsplit it is too many
// workgroups.
Plan plan_of(const Cache &c, int64_t n_heads, int64_t n_seqs, int64_t n_tokens, int64_t max_q, int64_t max_kv,
             int64_t window, int64_t sinks) {
    const int64_t rows = max_q * (n_heads / c.n_kv_heads), pairs = c.n_kv_heads * n_seqs;
    const double result_bytes = (double)(n_tokens * n_heads) * c.head_dim * 8;
    int64_t seen = max_kv;
    if (window && window + max_q + sinks < seen) seen = window + max_q + sinks;
    auto tiles = [&](int64_t tn) { return std::max((seen + tn - 1) / tn, (int64_t)1) + (window > 0); };
    auto blocks = [&](int64_t n) { return (rows + n - 1) / n; };
    const bool wide = c.head_dim > 128;
    Plan p;
    // More than 16 rows, but little to see and few enough blocks of 16: the few-row kernel has more workgroups
    // (prompts of 50, 100 and 200 tokens 7.5, 7.9 and 11.4 us; blocks of 64 rows 9.8, 11.5 and 13.8).  For 256
    // dimensions, where one workgroup fills a CU, up to one a CU (128 and 200 tokens 13.3 and 26.4 us, blocks of 64
    // rows 15.3 and 19.5).
    if (rows <= 16 || (tiles(32) <= 32 && blocks(16) * pairs <= (wide ? 256 : 512))) p.rows = 16;
    else if (wide) p.rows = 64;
    else if (rows <= 32) p.rows = 32;
    else if (rows <= 64) p.rows = 64;
    else p.rows = 128;
    double time = 0.0;
    int64_t per = 0;
    if (p.rows == 128) {
        per = many_per(tiles(64), blocks(128) * pairs, result_bytes, &time);
        // Blocks of 64 rows, 2.1 us a tile, where those of 128 leave CUs idle and it costs no more: prompts of 333,
        // 1000 and 2000 tokens 18.3, 39.4 and 87.3 us instead of 23.6, 54.3 and 100.7; of 3000 172.5, not 158.1.
        if (blocks(128) * pairs <= 512 &&
            2.1 * (double)tiles(64) * std::max(1.0, (double)(blocks(64) * pairs) / 512.0) <= time)
            p.rows = 64, per = tiles(64);
    }
    p.blocks = (int)blocks(p.rows);
    const int64_t n = tiles(p.few() || wide ? 32 : 64), grid = blocks(p.rows) * pairs;
    if (p.few()) per = few_per(n, grid, n_seqs);
    else if (per == 0) per = many_per(n, grid, result_bytes, &time);  // at most 64 rows
    if (grid > MAX_GROUPS) {
        p.rows = 0;
        return p;
    }
    const int64_t most = std::min((int64_t)MAX_SPLITS, MAX_GROUPS / grid);
    per = std::max(per, (n + most - 1) / most);
    p.per = (int)per;
    p.splits = (int)((n + per - 1) / per);
    // Prompts: their last blocks see most, and go first in every head (4096 tokens of 32 key-value heads 274 us, head
    // after head 348; eight ragged ones of up to 1000 with 8 and 4 heads 93 and 91, 100 and 95; but with one 109 and
    // 96).  Blocks of one window or of a chunk after a long cache see alike, and neighbours share what they read
    // (three windowed prompts 177 us head after head, 182).
    p.by_block = c.n_kv_heads % 4 == 0 && !window && 2 * max_q >= max_kv;
    // Many short sequences: one wave each, which starts alone and has no join (8 key-value heads of 128, 256 sequences
    // of 50, 100 and 300 tokens 13.3, 17.7 and 42.3 us, four waves 26.3, 27.7 and 46.9; 500 of 100 34.4 and 55.1; 128
    // of 100 and 500 12.3 and 36.5, 15.6 and 36.7; but 64 of 100 10.8 and 9.1).  For 256 dimensions a CU holds one
    // workgroup of four (64 of 50 and 200 12.8 and 21.9, 18.0 and 24.6).
    p.waves = p.rows == 16 && (n == 1 || (n <= 12 && grid >= (wide ? 512 : 1024))) ? 1 : 4;
    return p;
}

bool fine_sizes(const Cache &c, int64_t n_heads, int64_t n_seqs, int64_t n_tokens, int64_t max_q, int64_t max_kv,
                int64_t window, int64_t sinks) {
    return n_heads >= 1 && n_heads <= 65535 && n_heads % c.n_kv_heads == 0 && n_seqs >= 0 && n_seqs <= 65535 &&
           n_tokens >= 0 && n_tokens <= ((int64_t)1 << 23) && max_q >= 0 && max_q <= n_tokens && max_kv >= 0 &&
           max_kv <= MAX_LENGTH && window >= 0 && sinks >= 0 && window <= MAX_LENGTH && sinks <= MAX_LENGTH &&
           n_tokens * (n_heads / c.n_kv_heads) <= (1 << 30);
}

template <bool BF16, int DP, int DU, bool FULL>
int launch(const AttnArgs &a, const Plan &p, hipStream_t s) {
    const dim3 few((unsigned)(a.c.n_kv_heads * p.blocks * a.n_seqs * p.splits));
    const dim3 many((unsigned)(p.blocks * a.c.n_kv_heads * a.n_seqs), (unsigned)p.splits);
    if (p.rows == 16 && p.waves == 1) hipLaunchKernelGGL((few_kernel<BF16, DP, DU, FULL, 1, 1>), few, dim3(64), 0, s, a);
    else if (p.rows == 16) hipLaunchKernelGGL((few_kernel<BF16, DP, DU, FULL, 1, 4>), few, dim3(256), 0, s, a);
    else if (p.rows == 64) hipLaunchKernelGGL((many_kernel<BF16, DP, DU, FULL, 64>), many, dim3(256), 0, s, a);
    else if constexpr (DP < 256) {
        if (p.rows == 32) hipLaunchKernelGGL((few_kernel<BF16, DP, DU, FULL, 2, 4>), few, dim3(256), 0, s, a);
        else hipLaunchKernelGGL((many_kernel<BF16, DP, DU, FULL, 128>), many, dim3(256), 0, s, a);
    }
    return (int)hipGetLastError();
}

template <int TN, int ROWS, int LANES>
void launch_join(const AttnArgs &a, int64_t max_q, hipStream_t s) {
    const int64_t rows = max_q * a.group;
    if (a.splits <= SOME_SPLITS) {
        const dim3 grid((unsigned)((rows * LANES + 255) / 256), (unsigned)a.c.n_kv_heads, (unsigned)a.n_seqs);
        hipLaunchKernelGGL((join_some_kernel<TN, ROWS, LANES>), grid, dim3(256), 0, s, a);
    } else {
        const dim3 grid((unsigned)rows, (unsigned)a.c.n_kv_heads, (unsigned)a.n_seqs);
        hipLaunchKernelGGL((join_kernel<TN, ROWS, LANES>), grid, dim3(256), 0, s, a);
    }
}

template <int LANES>
void launch_join(const AttnArgs &a, int rows, int64_t max_q, hipStream_t s) {
    constexpr int DP = LANES * 4;
    if (rows == 16) launch_join<32, 16, LANES>(a, max_q, s);
    else if (rows == 64) launch_join<Many<DP, 64>::TN, 64, LANES>(a, max_q, s);
    else if constexpr (DP < 256) {
        if (rows == 32) launch_join<32, 32, LANES>(a, max_q, s);
        else launch_join<64, 128, LANES>(a, max_q, s);
    }
}

// 65 to 96 dimensions, and 129 to 192, take 3/4 of the matrix work of 128 and 256: prompts of 4096 tokens of 80 and of
// 160 dimensions 224 and 471 us in f16, 282 and 555 in bf16; with all of it 258 and 565, 333 and 667.
template <bool BF16>
int launch_dim(const AttnArgs &a, const Plan &p, hipStream_t s) {
    const int D = a.c.head_dim;
    if (D <= 64) return D == 64 ? launch<BF16, 64, 64, true>(a, p, s) : launch<BF16, 64, 64, false>(a, p, s);
    if (D <= 96) return launch<BF16, 128, 96, false>(a, p, s);
    if (D <= 128) return D == 128 ? launch<BF16, 128, 128, true>(a, p, s) : launch<BF16, 128, 128, false>(a, p, s);
    if (D <= 192) return launch<BF16, 256, 192, false>(a, p, s);
    return D == 256 ? launch<BF16, 256, 256, true>(a, p, s) : launch<BF16, 256, 256, false>(a, p, s);
}

}  // namespace

extern "C" size_t hip_qmm_attn_paged_workspace_size(const hip_qmm_kv_cache *cache, int64_t n_heads, int64_t n_seqs,
                                                    int64_t n_tokens, int64_t max_q, int64_t max_kv, int64_t window,
                                                    int64_t sinks) {
    Cache c;
    if (!take(cache, &c) || !fine_sizes(c, n_heads, n_seqs, n_tokens, max_q, max_kv, window, sinks) || max_q == 0 ||
        n_seqs == 0)
        return 0;
    const Plan p = plan_of(c, n_heads, n_seqs, n_tokens, max_q, max_kv, window, sinks);
    return p.rows == 0 || p.splits == 1 ? 0 : (size_t)p.splits * n_tokens * n_heads * (c.head_dim + 2) * sizeof(float);
}

extern "C" int hip_qmm_attn_paged_rows(const hip_qmm_kv_cache *cache, int64_t n_heads, int64_t n_seqs,
                                       int64_t n_tokens, int64_t max_q, int64_t max_kv, int64_t window, int64_t sinks,
                                       int *splits) {
    Cache c;
    if (!take(cache, &c) || !fine_sizes(c, n_heads, n_seqs, n_tokens, max_q, max_kv, window, sinks) || max_q == 0 ||
        n_seqs == 0)
        return 0;
    const Plan p = plan_of(c, n_heads, n_seqs, n_tokens, max_q, max_kv, window, sinks);
    if (splits && p.rows) *splits = p.splits;
    return p.rows;
}

extern "C" int hip_qmm_attn_paged(const hip_qmm_kv_cache *cache, const float *q, int64_t n_heads,
                                  int64_t q_token_stride, int64_t q_head_stride, const int32_t *q_starts,
                                  int64_t n_seqs, int64_t n_tokens, int64_t max_q, const int32_t *page_table,
                                  int64_t table_stride, const int32_t *kv_lens, int64_t max_kv, float scale,
                                  int64_t window, int64_t sinks, float *dst, int64_t dst_token_stride,
                                  int64_t dst_head_stride, void *workspace, size_t workspace_size, void *stream) {
    AttnArgs a = {};
    const int64_t lim = (int64_t)1 << 40;
    if (!take(cache, &a.c) || !fine_sizes(a.c, n_heads, n_seqs, n_tokens, max_q, max_kv, window, sinks) ||
        !isfinite(scale * LOG2E) || table_stride < 0 || table_stride > INT32_MAX)
        return (int)hipErrorInvalidValue;
    const int64_t H = a.c.n_kv_heads, D = a.c.head_dim;
    if (!q_starts && (n_tokens != n_seqs || (n_tokens > 0 && max_q < 1))) return (int)hipErrorInvalidValue;
    if (n_seqs == 0 || n_tokens == 0 || max_q == 0) return 0;
    if (!q || !dst || !kv_lens || (table_stride > 0 && !page_table)) return (int)hipErrorInvalidValue;
    if (((uintptr_t)q | (uintptr_t)dst) & 15 || ((q_token_stride | q_head_stride | dst_token_stride | dst_head_stride) & 3) ||
        q_token_stride < 0 || q_head_stride < 0 || dst_token_stride < 0 || dst_head_stride < 0 || q_token_stride > lim ||
        q_head_stride > lim || dst_token_stride > lim || dst_head_stride > lim || (n_heads > 1 && dst_head_stride < D) ||
        (n_tokens > 1 && dst_token_stride < (n_heads - 1) * dst_head_stride + D))
        return (int)hipErrorInvalidValue;
    const Plan p = plan_of(a.c, n_heads, n_seqs, n_tokens, max_q, max_kv, window, sinks);
    if (p.rows == 0) return (int)hipErrorInvalidValue;
    const int64_t rows = (int64_t)p.splits * n_tokens * n_heads;
    if (p.splits > 1 && (!workspace || ((uintptr_t)workspace & 15) ||
                         workspace_size < (size_t)rows * (D + 2) * sizeof(float)))
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
    a.n_tokens = (int)n_tokens;
    a.scale = scale * LOG2E;
    a.window = (int)window;
    a.sinks = (int)sinks;
    a.per = p.per;
    a.splits = p.splits;
    a.blocks = p.blocks;
    a.by_block = p.by_block;
    a.part_o = (float *)workspace;
    a.part_ml = (float *)workspace + rows * D;
    hipStream_t s = (hipStream_t)stream;
    const int e = cache->type == HIP_QMM_TYPE_BF16 ? launch_dim<true>(a, p, s) : launch_dim<false>(a, p, s);
    if (e || p.splits == 1) return e;
    if (D <= 64) launch_join<16>(a, p.rows, max_q, s);
    else if (D <= 128) launch_join<32>(a, p.rows, max_q, s);
    else launch_join<64>(a, p.rows, max_q, s);
    return (int)hipGetLastError();
}
