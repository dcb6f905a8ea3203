// i8_few.hip -- the 8-bit product for few columns: what counts is that the
// weights stream from memory without a pause.
//
// A workgroup of eight waves takes some weight rows, in blocks of 16, and up to 16 * NT
// columns.  (Row block, step of 128 inner bytes) are its items; wave w takes
// items w, w + 8, ..., each through a ring of its own in LDS that direct
// global->LDS transfers fill DEPTH items ahead: no barrier, and the next row
// block's weights are on their way while this one's are contracted.  Sums of a
// row block are collected in registers while the wave stays in it and then added
// to the workgroup's in LDS; integer sums do not depend on the order.
//
// The columns are in LDS whole (quantized there, if they come as f32), or come
// with the weights through the ring where they do not fit.  Their transfers are
// issued before the weights', and so are waited for without them.
//
// HBM bound: 14336 x 4096 by 24 columns take 14.2 us (4.2 TB/s of weights; a copy
// reaches 5.1), 4096 x 14336 by one 13.2 to 15; 48 tokens by 8 of 128 experts of
// 2048 x 768, f32, 36 to 45 (4.4 to 5.4 TB/s of the weights asked for).  What is
// short of the copy's rate is the start of a launch, with no transfer under way
// until the columns' rows are known, and its end.
#include <math.h>

#include <algorithm>

#include "i8.h"

using namespace i8;

namespace {

typedef __attribute__((address_space(3))) void *lds_ptr;

constexpr int WAVES = 8, THREADS = 64 * WAVES;
constexpr int STEP = 128;
constexpr int BLOCK = 16 * STEP;  // bytes of an item's weights

__device__ __forceinline__ uint32_t lds_addr(const void *p) { return (uint32_t)(uintptr_t)(lds_ptr)p; }

// 16 bytes per lane from its address to LDS at lds_base + 16 * lane (lds_base
// wave-uniform, in M0, whose write needs one wait state before it is read).
// Inline assembly, so that the compiler puts no vmcnt(0) of its own before LDS
// reads of other items; every wait is wait_for's.
__device__ __forceinline__ void dma16(const int8_t *from, uint32_t lds_base) {
    asm volatile("s_nop 0\n\tglobal_load_lds_dwordx4 %0, off" ::"v"(from), "{m0}"(lds_base) : "memory");
}

template <int N>
__device__ __forceinline__ void wait_for() {
    static_assert(N >= 0 && N <= 63, "vmcnt field");
    __builtin_amdgcn_s_waitcnt(0x0F70 | (N & 15) | ((N >> 4) << 14));
    asm volatile("" ::: "memory");
}

__device__ __forceinline__ void wait_reads() {
    __builtin_amdgcn_s_waitcnt(0xC07F);  // lgkmcnt(0)
    asm volatile("" ::: "memory");
}

struct Few {
    Product p;
    const int32_t *ids;     // by experts without a table: (token, slot) pairs
    int64_t ids_stride;
    int n_pairs, n_ids, n_as, per_slot;
    int rows;               // weight rows of a workgroup
    int x_bytes;            // of a column in LDS
    int columns;            // in LDS at once, at most 16 NT
    int staged;             // QUANTIZE: columns whose f32 values fit in LDS at once
    bool float4s;           // QUANTIZE: rows of whole aligned float4
};

// Chunk c of row r of 128 bytes sits at c ^ swizzle(r): the 16 rows that read one chunk column meet all banks.
__device__ __forceinline__ int swizzle(int r) { return (r >> 1) & 7; }

template <int NT, int DEPTH, FewMode MODE, bool IDS>
__global__ __launch_bounds__(THREADS) void few_kernel(Few f) {
    constexpr int PER = MODE == THROUGH ? 1 + NT : 1;  // 16-row blocks of an item in the ring
    const Product &a = f.p;
    extern __shared__ __attribute__((aligned(1024))) uint8_t smem[];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int r = lane & 15, g = lane >> 4;
    uint8_t *ring = smem + wave * (DEPTH * PER * BLOCK);
    int *sums = reinterpret_cast<int *>(smem + WAVES * DEPTH * PER * BLOCK);   // [blocks][NT][64 lanes][4]
    float *x_scale = reinterpret_cast<float *>(sums + (f.rows + 15) / 16 * NT * 256);  // [16 NT]
    int *src = reinterpret_cast<int *>(x_scale + 16 * NT), *dst = src + 16 * NT;
    int *found = dst + 16 * NT;                                                // [2 * WAVES]
    uint32_t *most = reinterpret_cast<uint32_t *>(found + 2 * WAVES);                // [WAVES]
    uint8_t *x_lds = reinterpret_cast<uint8_t *>(most + WAVES + 8);

    const int m0 = blockIdx.x * f.rows, m1 = min(m0 + f.rows, a.nrows), nb = (m1 - m0 + 15) / 16;
    const int8_t *w = a.w;
    const float *w_scale = a.w_scale;
    // Columns of this workgroup, or places among the expert's pairs.
    int first = IDS ? 0 : blockIdx.y * f.columns, end = IDS ? 0 : min(first + f.columns, a.ncols);
    int mine = 0;                  // IDS: the places of this thread's pair ...
    bool is = false;
    if constexpr (IDS) {
        // Workgroup y takes the y-th expert that some pair asks for; the last one clears the rows of ids that are no
        // expert's.
        const int own = tid < f.n_pairs ? f.ids[(int64_t)(tid / f.n_ids) * f.ids_stride + tid % f.n_ids] : -1;
        const bool valid = (uint32_t)own < (uint32_t)f.n_as;
        unsigned *asked = reinterpret_cast<unsigned *>(smem);  // a bit for each expert
        if (tid < 32) asked[tid] = 0;
        if (tid == 0) found[0] = -1;
        __syncthreads();
        if (blockIdx.y == gridDim.y - 1) {
            unsigned long long *bad = reinterpret_cast<unsigned long long *>(smem);
            const unsigned long long who = __ballot(tid < f.n_pairs && !valid);
            if (lane == 0) bad[wave] = who;
            __syncthreads();
            for (int v = 0; v < WAVES; ++v)
                for (unsigned long long rest = bad[v]; rest; rest &= rest - 1) {
                    float *out = a.dst + (int64_t)(v * 64 + __ffsll((long long)rest) - 1) * a.dst_stride;
                    for (int m = m0 + tid; m < m1; m += THREADS) out[m] = 0.0f;
                }
            return;
        }
        if (valid) atomicOr(&asked[own >> 5], 1u << (own & 31));
        __syncthreads();
        if (wave == 0) {
            const unsigned bits = lane < 32 ? asked[lane] : 0;
            int before = __popc(bits);
#pragma unroll
            for (int d = 1; d < 32; d <<= 1) {
                const int u = __shfl_up(before, d);
                if (lane >= d) before += u;
            }
            before -= __popc(bits);
            const int nth = (int)blockIdx.y - before;
            if (nth >= 0 && nth < __popc(bits)) {
                unsigned rest = bits;
                for (int i = 0; i < nth; ++i) rest &= rest - 1;
                found[0] = lane * 32 + __ffs(rest) - 1;
            }
        }
        __syncthreads();
        const int e = found[0];
        __syncthreads();
        if (e < 0) return;
        is = own == e;
        const unsigned long long who = __ballot(is);
        if (lane == 0) found[wave] = __popcll(who);
        __syncthreads();
        end = 0;
        for (int v = 0; v < WAVES; ++v) {
            if (v < wave) mine += found[v];
            end += found[v];
        }
        mine += __popcll(who & ((1ull << lane) - 1));
        w += (int64_t)e * a.expert_stride;
        w_scale += (int64_t)e * a.nrows;
    }

    const int steps = (a.K + STEP - 1) / STEP, items = nb * steps, tail = a.K - (steps - 1) * STEP;
    const int last_chunk = (tail - 1) >> 4;
    do {
        const int n = min(end - first, f.columns);
        // Which columns: rows of x and of the result.
        if constexpr (IDS) {
            if (is && mine >= first && mine < first + n) {
                src[mine - first] = f.per_slot ? tid : tid / f.n_ids;
                dst[mine - first] = tid;
            }
        } else {
            if (tid < n) src[tid] = dst[tid] = first + tid;
        }
        for (int i = tid; i < nb * NT * 256; i += THREADS) sums[i] = 0;
        __syncthreads();

        // The wave's next item into a slot of its ring; past the end 16 bytes of the first row, so that it can always wait
        // for the same number of transfers.
        int next_b = wave / steps, next_s = wave - next_b * steps;
        const int8_t *x_from[2 * NT];
        if constexpr (MODE == THROUGH) {
#pragma unroll
            for (int j = 0; j < 2 * NT; ++j)
                x_from[j] = a.x + (int64_t)src[min(8 * j + (lane >> 3), n - 1)] * a.x_stride;
        }
        auto bring = [&](int slot) {
            const int b = next_b, s = next_s;
            const bool real = b < nb;
            const uint32_t to = lds_addr(ring) + slot * (PER * BLOCK);
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int row = 8 * h + (lane >> 3);
                int chunk = (lane & 7) ^ swizzle(row);
                if (s == steps - 1) chunk = min(chunk, last_chunk);
                const int8_t *from = w + (int64_t)min(m0 + b * 16 + row, m1 - 1) * a.w_stride + s * STEP + chunk * 16;
                dma16(real ? from : w, to + h * 1024);
            }
            if constexpr (MODE == THROUGH) {
#pragma unroll
                for (int j = 0; j < 2 * NT; ++j) {
                    int chunk = (lane & 7) ^ swizzle(8 * j + (lane >> 3));
                    if (s == steps - 1) chunk = min(chunk, last_chunk);
                    dma16(real ? x_from[j] + s * STEP + chunk * 16 : a.x, to + BLOCK + j * 1024);
                }
            }
            next_s += WAVES;
            while (next_s >= steps) next_s -= steps, ++next_b;
        };
        auto bring_first = [&]() {
#pragma unroll
            for (int d = 0; d < DEPTH; ++d) bring(d);
        };
        // Bytes of columns c0 .. c0 + count, `bytes` of each, to rows of `stride` in LDS.
        auto bring_columns = [&](const uint8_t *from, int64_t from_stride, int c0, int count, int bytes, uint8_t *to, int stride) {
            const int parts = (bytes + 1023) / 1024;
            for (int i = wave; i < count * parts; i += WAVES) {
                const int c = i / parts, at = (i - c * parts) * 1024;
                if (at + lane * 16 < bytes)
                    dma16((const int8_t *)from + src[c0 + c] * from_stride + at + lane * 16, lds_addr(to) + c * stride + at);
            }
        };
        if constexpr (MODE == QUANTIZE) {
            uint8_t *stage = x_lds + f.columns * f.x_bytes;
            // Waves that share a column.
            const int units = (a.K + 3) / 4;  // float4
            const int share = n == 1 ? 8 : n == 2 ? 4 : n <= 4 ? 2 : 1, team = wave / share;
            for (int c0 = 0; c0 < n; c0 += f.staged) {
                const int count = min(f.staged, n - c0);
                if (f.float4s) {
                    bring_columns((const uint8_t *)a.x, a.x_stride * 4, c0, count, a.K * 4, stage, units * 16);
                } else {
                    for (int i = wave; i < count; i += WAVES) {
                        const float *row = (const float *)a.x + src[c0 + i] * a.x_stride;
                        float *to = reinterpret_cast<float *>(stage) + i * units * 4;
#pragma unroll 4
                        for (int k = lane * 4; k + 4 <= a.K; k += 256) *reinterpret_cast<float4 *>(to + k) = four_at(row + k);
                        if (const int k = a.K / 4 * 4 + lane; k < units * 4) to[k] = k < a.K ? row[k] : 0.0f;
                    }
                }
                if (c0 == 0) {
                    bring_first();
                    wait_for<2 * PER * DEPTH>();
                } else {
                    wait_for<0>();
                }
                __syncthreads();
                for (int base = 0; base < count; base += WAVES / share) {
                    const int c = base + team;
                    const float4 *row = reinterpret_cast<const float4 *>(stage + min(c, count - 1) * units * 16);
                    const int begin = tid - team * share * 64, hop = share * 64;
                    uint32_t m = 0;
                    for (int k = begin; k < units; k += hop) {
                        const float4 v = row[k];
                        m = max(m, max(max(magnitude(v.x), magnitude(v.y)), max(magnitude(v.z), magnitude(v.w))));
                    }
#pragma unroll
                    for (int d = 32; d; d >>= 1) m = max(m, (uint32_t)__shfl_xor((int)m, d));
                    if (share > 1) {
                        if (lane == 0) most[wave] = m;
                        __syncthreads();
                        for (int v = 0; v < share; ++v) m = max(m, most[team * share + v]);
                        __syncthreads();
                    }
                    const Scale scale(m);
                    if (c < count) {
                        for (int k = begin; k < units; k += hop)
                            *reinterpret_cast<uint32_t *>(x_lds + (c0 + c) * f.x_bytes + k * 4) = scale.four(row[k]);
                        if (begin == 0) x_scale[c0 + c] = scale.value;
                    }
                }
                __syncthreads();
            }
        } else {
            if (tid < n) x_scale[tid] = a.x_scale[src[tid]];
            if constexpr (MODE == RESIDENT)
                bring_columns((const uint8_t *)a.x, a.x_stride, 0, n, (a.K + 15) / 16 * 16, x_lds, f.x_bytes);
            bring_first();
            wait_for<2 * PER * DEPTH>();
            __syncthreads();
        }

        v4i acc[NT];
#pragma unroll
        for (int j = 0; j < NT; ++j) acc[j] = (v4i){};
        const uint8_t *x_row[NT];
#pragma unroll
        for (int j = 0; j < NT; ++j) x_row[j] = x_lds + min(16 * j + r, n - 1) * f.x_bytes + g * 16;
        const int at0 = r * STEP + ((g ^ swizzle(r)) << 4), at1 = r * STEP + (((4 + g) ^ swizzle(r)) << 4);
        int slot = 0, b = wave / steps, s = wave - b * steps;
        for (int i = wave; i < items; i += WAVES) {
            wait_for<2 * PER *(DEPTH - 1)>();
            const uint8_t *here = ring + slot * (PER * BLOCK);
            v4i u[2], v[2][NT];
            u[0] = *reinterpret_cast<const v4i *>(here + at0);
            u[1] = *reinterpret_cast<const v4i *>(here + at1);
#pragma unroll
            for (int j = 0; j < NT; ++j) {
                if constexpr (MODE == THROUGH) {
                    v[0][j] = *reinterpret_cast<const v4i *>(here + (1 + j) * BLOCK + at0);
                    v[1][j] = *reinterpret_cast<const v4i *>(here + (1 + j) * BLOCK + at1);
                } else {
                    v[0][j] = *reinterpret_cast<const v4i *>(x_row[j] + s * STEP);
                    v[1][j] = *reinterpret_cast<const v4i *>(x_row[j] + s * STEP + 64);
                }
            }
            wait_reads();
            bring(slot);
            if (s == steps - 1) {
                u[0] = cut(u[0], tail - g * 16);
                u[1] = cut(u[1], tail - 64 - g * 16);
            }
#pragma unroll
            for (int j = 0; j < NT; ++j) {
                acc[j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(u[0], v[0][j], acc[j], 0, 0, 0);
                acc[j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(u[1], v[1][j], acc[j], 0, 0, 0);
            }
            slot = slot + 1 == DEPTH ? 0 : slot + 1;
            const int was = b;
            s += WAVES;
            while (s >= steps) s -= steps, ++b;
            if (b != was) {
#pragma unroll
                for (int j = 0; j < NT; ++j) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) atomicAdd(sums + (was * NT + j) * 256 + e * 64 + lane, acc[j][e]);
                    acc[j] = (v4i){};
                }
            }
        }
        wait_for<0>();
        __syncthreads();

        // Column c, row m: 16 rows of a column side by side.
        for (int i = tid; i < n * nb * 16; i += THREADS) {
            const int c = i / (nb * 16), q = i - c * (nb * 16), m = m0 + q;
            if (m >= m1) continue;
            const int sum = sums[((q >> 4) * NT + (c >> 4)) * 256 + (q & 3) * 64 + ((q & 15) >> 2) * 16 + (c & 15)];
            a.dst[(int64_t)dst[c] * a.dst_stride + m] = scaled(sum, x_scale[c], w_scale[m]);
        }
        first += f.columns;
        if (first < end) __syncthreads();
    } while (IDS && first < end);
}

constexpr int LDS = 160 * 1024, HALF = LDS / 2;

// Bytes of a column in LDS: whole steps, and 16 more so that columns meet different banks.
int column_bytes(int64_t K) { return (int)((K + STEP - 1) / STEP * STEP + 16); }

int fixed_bytes(int nt, int depth, bool through, int rows) {
    return WAVES * depth * (through ? 1 + nt : 1) * BLOCK + (rows + 15) / 16 * nt * 1024 + 16 * nt * 12 + 2 * WAVES * 4 +
           (WAVES + 8) * 4;
}

// The plan's bytes of LDS, if at most `most`, with as many f32 columns staged as fit.
bool fits(FewPlan &p, int64_t K, int most) {
    int64_t bytes = fixed_bytes(p.nt, p.depth, p.mode == THROUGH, p.rows);
    if (p.mode != THROUGH) bytes += (int64_t)p.columns * column_bytes(K);
    if (p.mode == QUANTIZE) {
        p.staged = (int)std::min((int64_t)p.columns, std::max((int64_t)0, most - bytes) / ((K + 3) / 4 * 16));
        if (p.staged < 1) return false;
        bytes += p.staged * ((K + 3) / 4 * 16);
    }
    if (bytes > most) return false;
    p.bytes = (int)bytes;
    return true;
}

Few arguments(const Product &p, const FewPlan &plan) {
    Few f = {};
    f.float4s = !(p.K % 4 || p.x_stride % 4 || (uintptr_t)p.x % 16);
    f.p = p, f.rows = plan.rows, f.x_bytes = column_bytes(p.K), f.columns = plan.columns, f.staged = plan.staged;
    return f;
}

template <int NT, int DEPTH, FewMode MODE, bool IDS>
int launch(const Few &f, dim3 grid, int bytes, hipStream_t s) {
    hipLaunchKernelGGL((few_kernel<NT, DEPTH, MODE, IDS>), grid, dim3(THREADS), bytes, s, f);
    return (int)hipGetLastError();
}

}  // namespace

// Up to 32 columns: two workgroups a CU, two items ahead, where both fit and there are 16 rows for each: one's start
// overlaps the other's work (14336 x 4096 by one column 13.6 us, 14.2 with one a CU and four ahead); else one with as many
// items ahead as fit.  At least 8 rows, of the 16 that an instruction takes: fewer do not make a small product faster.
//
// More columns, 32 to a workgroup, where one round of workgroups takes them all: eight shares of K in each instead of a
// tile's long way along it on few CUs (1024 x 4096 by 64 columns 5.8 us, 10.2 in tiles; 269 x 16070 by 469 17.9, 30.5;
// 4096 x 4096 by 64, 32 rows a workgroup, 9.6, 10.8; with two rounds 524 x 4915 by 450 takes 13.7, 12.1 in tiles).
FewPlan i8::few_plan(bool f32, int64_t K, int64_t nrows, int64_t ncols) {
    FewPlan p = {};
    if (ncols < 1 || (f32 && ncols > 32)) return p;
    if (ncols > 32) {
        p.mode = THROUGH, p.nt = 2, p.depth = 3, p.columns = 32;
        for (p.rows = 16; p.rows <= 32; p.rows += 16)
            if ((nrows + p.rows - 1) / p.rows * ((ncols + 31) / 32) <= 256 && fits(p, K, LDS)) break;
        return p;
    }
    p.nt = ncols <= 16 ? 1 : 2;
    p.columns = (int)ncols;
    p.mode = f32 ? QUANTIZE : RESIDENT;
    // Every workgroup quantizes for itself, which costs more than a launch before it beyond some values.
    if (f32 && (ncols > 16 || (ncols > 1 && ncols * K > 16384))) return p;
    p.depth = 2;
    p.rows = (int)std::min((nrows + 511) / 512, (int64_t)256);
    if (p.rows >= 16 && fits(p, K, HALF)) return p;
    p.rows = (int)std::min(std::max((nrows + 255) / 256, (int64_t)8), (int64_t)256);
    for (p.depth = p.nt == 1 ? 4 : 3; p.depth >= 2; --p.depth)
        if ((p.depth != 3 || p.nt == 2) && fits(p, K, LDS)) return p;
    if (f32) return p;
    p.mode = THROUGH;
    p.depth = p.nt == 1 ? 4 : 3;
    fits(p, K, LDS);
    return p;
}

// At most 512 pairs, and on the average at most 12 of an expert.  Two workgroups a CU, as many rows each as make 512 of
// them if every pair asks for another expert.
FewPlan i8::few_pairs_plan(bool f32, int64_t K, int64_t nrows, int64_t n_as, int64_t n_tokens, int64_t n_ids) {
    FewPlan p = {};
    const int64_t pairs = n_tokens * n_ids, experts = std::min(pairs, n_as);
    if (pairs > THREADS || pairs > 12 * experts) return p;
    // Workgroups of other experts and rows quantize the same tokens (128 experts of 1536 x 2048: 8 tokens 31.7 us, 34.3 with a
    // launch before; 16 tokens 62.4, 52.1).
    if (f32 && n_tokens > 1 && n_tokens * K > 16384) return p;
    p.mode = f32 ? QUANTIZE : RESIDENT;
    p.nt = 1;
    p.depth = 2;
    p.columns = (int)std::min(n_tokens, (int64_t)16);  // of an expert, unless a token asks for it twice
    const int64_t want = std::min((experts * nrows + 511) / 512, std::min(nrows, (int64_t)512));
    const int rows = (int)std::max((want + 15) / 16 * 16, (int64_t)16), least = std::min(rows, 64);
    for (const int most : {HALF, LDS})
        for (p.rows = rows; p.rows >= least; p.rows -= 16)
            if (fits(p, K, most) && (!f32 || p.staged >= std::min(p.columns, 2))) return p;
    if (f32 && n_tokens > 1) return p = {};
    // Long rows: fewer columns at a time, and the weights read again for the others.
    for (p.rows = least; p.columns > 4; --p.columns)
        if (fits(p, K, LDS)) return p;
    fits(p, K, LDS);
    return p;
}

int i8::few_product(const Product &p, const FewPlan &plan, hipStream_t s) {
    const dim3 grid((unsigned)((p.nrows + plan.rows - 1) / plan.rows), (unsigned)((p.ncols + plan.columns - 1) / plan.columns));
    const Few f = arguments(p, plan);
#define FEW(NT, DEPTH, MODE) \
    if (plan.nt == NT && plan.depth == DEPTH && plan.mode == MODE) return launch<NT, DEPTH, MODE, false>(f, grid, plan.bytes, s)
    FEW(1, 4, QUANTIZE);
    FEW(1, 2, QUANTIZE);
    FEW(1, 4, RESIDENT);
    FEW(1, 2, RESIDENT);
    FEW(2, 3, RESIDENT);
    FEW(2, 2, RESIDENT);
    FEW(1, 4, THROUGH);
    FEW(2, 3, THROUGH);
#undef FEW
    return (int)hipErrorInvalidValue;
}

int i8::few_pairs(const Product &p, const FewPlan &plan, const int32_t *ids, int64_t ids_stride, int n_pairs, int n_ids,
                  int n_as, int per_slot, hipStream_t s) {
    Few f = arguments(p, plan);
    f.ids = ids, f.ids_stride = ids_stride, f.n_pairs = n_pairs, f.n_ids = n_ids, f.n_as = n_as, f.per_slot = per_slot;
    const dim3 grid((unsigned)((p.nrows + plan.rows - 1) / plan.rows), (unsigned)std::min(n_pairs, n_as) + 1);
    return plan.mode == QUANTIZE ? launch<1, 2, QUANTIZE, true>(f, grid, plan.bytes, s)
                                 : launch<1, 2, RESIDENT, true>(f, grid, plan.bytes, s);
}
