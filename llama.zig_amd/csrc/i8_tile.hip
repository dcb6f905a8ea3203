// i8_tile.hip -- the 8-bit product for many columns: tiles of weights and
// columns in LDS, contracted on 32x32x32 integer matrix instructions.
//
// Four waves, two by two, share a tile of TM weight rows and TN columns.  The
// inner axis goes by in stages of 128 bytes, which direct global->LDS transfers
// bring into two rings, SW stages of weights and SX of columns; a stage is four
// steps of 32 bytes, and the operands of a unit of G steps are read from LDS
// while the unit before is contracted.  One barrier a stage: before its last unit
// is contracted, whose operands are in registers by then, so that the stage's
// places are free.  The transfers into them are issued among the matrix
// instructions from there on: all at once they would wait for each other.
//
// 14336 x 4096 by 4096 columns, 256 x 256 tiles: 228 us, 2.11 POP/s (a library's
// product of these sizes 226, of 8192^3 2.44 POP/s).  A tile's stages run at 78 % of
// the matrix cycles of a clock that falls to 1.63 to 1.7 GHz under them; its first
// transfers take 2.5 us and its results 9 to 11 of 62.  Small tiles (5003 x 2720 by 333, 128 x 64:
// 14.5 us) are bound by reading operands from L2, 11 to 14 TB/s in all.
#include <algorithm>

#include "i8.h"

using namespace i8;

namespace {

typedef int v16i __attribute__((ext_vector_type(16)));
typedef __attribute__((address_space(3))) void *lds_ptr;

constexpr int STAGE = 128;  // bytes of the inner axis

__device__ __forceinline__ uint32_t lds_addr(const void *p) { return (uint32_t)(uintptr_t)(lds_ptr)p; }

// 16 bytes per lane from its address to LDS at lds_base + 16 * lane (lds_base
// wave-uniform, in M0, whose write needs one wait state before it is read).
// Inline assembly, so that the compiler, which cannot tell the stages of the
// ring apart, puts no vmcnt(0) of its own before the LDS reads of another stage;
// every wait is wait_for's.
__device__ __forceinline__ void dma16(const int8_t *from, uint32_t lds_base) {
    asm volatile("s_nop 0\n\tglobal_load_lds_dwordx4 %0, off" ::"v"(from), "{m0}"(lds_base) : "memory");
}

// All LDS reads, and all but the last N transfers.
template <int N>
__device__ __forceinline__ void wait_for() {
    static_assert(N >= 0 && N <= 63, "vmcnt field");
    __builtin_amdgcn_s_waitcnt(0x0070 | (N & 15) | ((N >> 4) << 14));
    asm volatile("" ::: "memory");
}

__device__ __forceinline__ void barrier() {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
}

// A tile's row of 128 bytes is 8 chunks; chunk c of row r sits at c ^ swizzle(r), so that the 16 rows that read one
// chunk column together meet all banks.
__device__ __forceinline__ int swizzle(int r) { return (r >> 1) & 7; }

// A tile's work: TM weight rows from m0 and TN columns from `first`, before `end`.
template <int TM, int TN, int SW, int SX, int G>
__device__ __forceinline__ void tile(const Product &a, uint8_t *ring, const int8_t *w, const float *w_scale, int m0,
                                     int first, int end) {
    constexpr int RM = TM / 64, RN = TN / 64;            // 32 x 32 tiles of a wave
    constexpr int LM = TM / 32, LN = TN / 32, L = LM + LN;  // transfers of a wave and stage
    constexpr int WB = TM * STAGE, XB = TN * STAGE, XRING = SW * WB;
    // A unit is G steps; the products of one, its operands' reads, one after each product if there are as many products.
    constexpr int UNITS = 4 / G, PRODUCTS = G * RM * RN, READS = G * (RM + RN), SLOTS = READS < PRODUCTS ? PRODUCTS : READS;
    constexpr int TOGETHER = UNITS > 1 ? 1 : 2;  // stages of a loop's turn, so that the operands' two sets take turns
    static_assert(UNITS > 1 || SW == SX, "one unit: the transfers of a stage are issued together");
    static_assert(SW >= SX && SX >= 2 && TM <= 256 && TN <= 256, "rings and scales");
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wm = wave >> 1, wn = wave & 1;
    w += (int64_t)m0 * a.w_stride;

    // Transfer i of the wave: 8 rows, a lane 16 bytes of row lane / 8.  The weights' come first.
    const int8_t *from[L];
#pragma unroll
    for (int i = 0; i < L; ++i) {
        const bool of_w = i < LM;
        const int row = 8 * (of_w ? wave * LM + i : wave * LN + i - LM) + (lane >> 3);
        const int chunk = (lane & 7) ^ swizzle(row);
        if (of_w) {
            from[i] = w + (int64_t)min(row, a.nrows - 1 - m0) * a.w_stride + chunk * 16;
        } else {
            const int c = min(first + row, end - 1);
            from[i] = a.x + (int64_t)(a.tiles ? a.col_src[c] : c) * a.x_stride + chunk * 16;
        }
    }
    // The tile's scales and result rows, for the end.
    const int own_c = min(first + (int)threadIdx.x, end - 1);
    const float own_w = w_scale[min(m0 + (int)threadIdx.x, a.nrows - 1)];
    const float own_x = a.x_scale[a.tiles ? a.col_src[own_c] : own_c];
    const int own_row = a.tiles ? a.col_dst[own_c] : own_c;

    const int whole = a.K / STAGE, tail = a.K - whole * STAGE, stages = whole + (tail > 0);
    const uint32_t lds = lds_addr(ring);
    auto transfer = [&](int t, int i, int step) {
        dma16(from[i], i < LM ? lds + (uint32_t)(t % SW) * WB + (wave * LM + i) * 1024
                              : lds + XRING + (uint32_t)(t % SX) * XB + (wave * LN + i - LM) * 1024);
        from[i] += step;
    };
    // Before stage t of transfers lo..hi: in the stage that K ends in, chunks past the end repeat its last chunk.
    // Behind the last stage the transfers go on, so that there is one loop and one count to wait for, but of 16 bytes
    // of the first row for all lanes.
    auto turn_to = [&](int t, int lo, int hi) {
        if (t == whole && tail) {
            const int last = (tail - 1) >> 4;
#pragma unroll
            for (int i = 0; i < L; ++i)
                if (i >= lo && i < hi) {
                    const int chunk = (lane & 7) ^ swizzle(8 * (i < LM ? wave * LM + i : wave * LN + i - LM) + (lane >> 3));
                    from[i] -= max(chunk - last, 0) * 16;
                }
        }
        if (t >= stages) {
#pragma unroll
            for (int i = 0; i < L; ++i)
                if (i >= lo && i < hi) from[i] = w;
        }
    };

    // Where the lane reads chunk 2 s + lane / 32 of its rows.
    const int r = lane & 31, h = lane >> 5;
    int read[4];
#pragma unroll
    for (int s = 0; s < 4; ++s) read[s] = r * STAGE + (((2 * s + h) ^ swizzle(r)) << 4);
    const uint8_t *at_w = ring + wm * (TM / 2) * STAGE, *at_x = ring + XRING + wn * (TN / 2) * STAGE;
    v4i fw[2][G][RM], fx[2][G][RN];
    auto read_w = [&](int t, int s, int i) {
        return *reinterpret_cast<const v4i *>(at_w + (t % SW) * WB + read[s] + i * 32 * STAGE);
    };
    auto read_x = [&](int t, int s, int j) {
        return *reinterpret_cast<const v4i *>(at_x + (t % SX) * XB + read[s] + j * 32 * STAGE);
    };

    v16i acc[RM][RN];
#pragma unroll
    for (int i = 0; i < RM; ++i)
#pragma unroll
        for (int j = 0; j < RN; ++j) acc[i][j] = (v16i){};

    // The first stages, in the order in which they go on below.
#pragma unroll
    for (int t = 0; t < SW; ++t) {
        if (t < SX) {
            turn_to(t, LM, L);
#pragma unroll
            for (int i = LM; i < L; ++i) transfer(t, i, STAGE);
        }
        if (t < SW - (UNITS > 1)) {
            turn_to(t, 0, LM);
#pragma unroll
            for (int i = 0; i < LM; ++i) transfer(t, i, STAGE);
        }
    }
    wait_for<L *(SX - 1) + (SW == SX && UNITS > 1 ? -LM : 0) + LM *(SW > SX ? SW - SX - 1 : 0)>();
    barrier();
    // Operand l of a unit, in the order in which it needs them.
    auto fetch = [&](int buffer, int t, int unit, int l) {
        const int q = l / (RM + RN), o = l % (RM + RN), s = unit * G + q;
        if (o == 0)
            fw[buffer][q][0] = read_w(t, s, 0);
        else if (o <= RN)
            fx[buffer][q][o - 1] = read_x(t, s, o - 1);
        else
            fw[buffer][q][o - RN] = read_w(t, s, o - RN);
    };
#pragma unroll
    for (int l = 0; l < READS; ++l) fetch(0, 0, 0, l);

#pragma clang loop unroll(disable)
    for (int t0 = 0; t0 < whole; t0 += TOGETHER) {
#pragma unroll
        for (int v = 0; v < TOGETHER; ++v) {
            const int t = t0 + v;
            if (v > 0 && t >= whole) break;
#pragma unroll
            for (int s = 0; s < UNITS; ++s) {
                const bool last = s == UNITS - 1;
                const int now = (TOGETHER > 1 ? v : s) & 1;
                if (last) {
                    // Stage t is in registers, and stage t + 1 in LDS.
                    wait_for<L *(SX - 2) + (SW > SX ? LM : 0)>();
                    barrier();
                    turn_to(t + SX, LM, L);
                }
                // Transfers go into the places of the last stage that is done with: the columns' from here on, the
                // weights' in the unit after.
                const int weights = UNITS > 1 ? t - 1 : t;
                if (s == 0) turn_to(weights + SW, 0, LM);
#pragma unroll
                for (int k = 0; k < PRODUCTS; ++k) {
                    const int q = k / (RM * RN), i = k / RN % RM, j = k % RN;
                    acc[i][j] = __builtin_amdgcn_mfma_i32_32x32x32_i8(fw[now][q][i], fx[now][q][j], acc[i][j], 0, 0, 0);
                    // What goes on beside the matrix instructions, little after each: the next unit's operands, and the
                    // transfers.
#pragma unroll
                    for (int l = k * SLOTS / PRODUCTS; l < (k + 1) * SLOTS / PRODUCTS; ++l)
                        if (l < READS) fetch(now ^ 1, last ? t + 1 : t, last ? 0 : s + 1, l);
#pragma unroll
                    for (int l = k * LN / PRODUCTS; l < (k + 1) * LN / PRODUCTS; ++l)
                        if (last) transfer(t + SX, LM + l, STAGE);
#pragma unroll
                    for (int l = k * LM / PRODUCTS; l < (k + 1) * LM / PRODUCTS; ++l)
                        if (s == 0) transfer(weights + SW, l, STAGE);
                    __builtin_amdgcn_sched_barrier(0);
                }
            }
        }
    }
    if (tail) {
        for (int s = 0; s * 32 < tail; ++s) {
            v4i u[RM];
            const int at = r * STAGE + (((2 * s + h) ^ swizzle(r)) << 4);
#pragma unroll
            for (int i = 0; i < RM; ++i)
                u[i] = cut(*reinterpret_cast<const v4i *>(at_w + whole % SW * WB + at + i * 32 * STAGE), tail - (2 * s + h) * 16);
#pragma unroll
            for (int j = 0; j < RN; ++j) {
                const v4i v = *reinterpret_cast<const v4i *>(at_x + whole % SX * XB + at + j * 32 * STAGE);
#pragma unroll
                for (int i = 0; i < RM; ++i) acc[i][j] = __builtin_amdgcn_mfma_i32_32x32x32_i8(u[i], v, acc[i][j], 0, 0, 0);
            }
        }
    }

    // Results go out through LDS, 32 columns of each wave at a time, so that stores are of whole rows of the tile and
    // the code is small (unrolled over the accumulators it took 20 us to fetch).  Lane (r, h) has column r and rows
    // 8 q + 4 h + {0..3} of each 32 x 32; in LDS 4 rows are a chunk, and chunk c of column r sits at c ^ (r & 15).
    constexpr int CHUNKS = TM / 8, COLS = 64 / CHUNKS;  // chunks of a wave's column, columns of a store
    constexpr int AT_ONCE = 32 / COLS < 8 ? 32 / COLS : 8;
    static_assert(32 % (COLS * AT_ONCE) == 0, "whole rounds of 32 columns");
    wait_for<0>();
    barrier();
    float *scales = reinterpret_cast<float *>(ring + 4 * 32 * CHUNKS * 16);
    int *rows = reinterpret_cast<int *>(scales + TM + TN);
    if (threadIdx.x < TM) scales[threadIdx.x] = own_w;
    if (threadIdx.x < TN) scales[TM + threadIdx.x] = own_x, rows[threadIdx.x] = own_row;
    const bool moderate_ones = __all(moderate(own_w) && moderate(own_x));
    if (lane == 0) rows[TN + wave] = moderate_ones;
    __syncthreads();
    const bool plain = rows[TN] && rows[TN + 1] && rows[TN + 2] && rows[TN + 3];
    v4i *turn = reinterpret_cast<v4i *>(ring) + wave * 32 * CHUNKS;
    const int mine = lane % CHUNKS * 4, m = m0 + wm * (TM / 2) + mine, left = a.nrows - m;
    const float4 ws = *reinterpret_cast<const float4 *>(scales + wm * (TM / 2) + mine);
    const bool whole_tile = first + TN <= end && m0 + TM <= a.nrows;
    typedef float v4f __attribute__((ext_vector_type(4), aligned(4)));  // a store of 16 bytes need not be aligned
    float *const out = a.dst + m;
#pragma clang loop unroll(disable)
    for (int j = 0; j < RN; ++j) {
#pragma unroll
        for (int jj = 0; jj < RN; ++jj)
            if (j == jj) {
#pragma unroll
                for (int i = 0; i < RM; ++i)
#pragma unroll
                    for (int q = 0; q < 4; ++q)
                        turn[r * CHUNKS + ((8 * i + 2 * q + h) ^ (r & (CHUNKS - 1) & 15))] =
                            (v4i){acc[i][jj][4 * q], acc[i][jj][4 * q + 1], acc[i][jj][4 * q + 2], acc[i][jj][4 * q + 3]};
            }
        const int c0 = wn * (TN / 2) + j * 32;
#pragma clang loop unroll(disable)
        for (int k = 0; k < 32; k += COLS * AT_ONCE) {
            v4i s[AT_ONCE];
            float xs[AT_ONCE];
            int row[AT_ONCE];
#pragma unroll
            for (int u = 0; u < AT_ONCE; ++u) {
                const int c = k + u * COLS + lane / CHUNKS;
                s[u] = turn[c * CHUNKS + (lane % CHUNKS ^ (c & (CHUNKS - 1) & 15))];
                xs[u] = scales[TM + c0 + c];
                row[u] = rows[c0 + c];
            }
            if (plain && whole_tile) {
#pragma unroll
                for (int u = 0; u < AT_ONCE; ++u)
                    *reinterpret_cast<v4f *>(out + (int64_t)row[u] * a.dst_stride) =
                        (v4f){(float)s[u][0] * xs[u] * ws.x, (float)s[u][1] * xs[u] * ws.y, (float)s[u][2] * xs[u] * ws.z,
                              (float)s[u][3] * xs[u] * ws.w};
            } else {
#pragma unroll
                for (int u = 0; u < AT_ONCE; ++u) {
                    if (first + c0 + k + u * COLS + lane / CHUNKS >= end) continue;
                    float *o = out + (int64_t)row[u] * a.dst_stride;
                    const v4f v = plain ? (v4f){(float)s[u][0] * xs[u] * ws.x, (float)s[u][1] * xs[u] * ws.y,
                                                (float)s[u][2] * xs[u] * ws.z, (float)s[u][3] * xs[u] * ws.w}
                                        : (v4f){scaled(s[u][0], xs[u], ws.x), scaled(s[u][1], xs[u], ws.y),
                                                scaled(s[u][2], xs[u], ws.z), scaled(s[u][3], xs[u], ws.w)};
                    if (left >= 4) {
                        *reinterpret_cast<v4f *>(o) = v;
                    } else {
                        if (left > 0) o[0] = v[0];
                        if (left > 1) o[1] = v[1];
                        if (left > 2) o[2] = v[2];
                    }
                }
            }
        }
    }
}

constexpr int NEIGHBOURS = 32;  // CUs of an XCD

template <int TM, int TN, int SW, int SX, int G, bool HALVES>
__global__ __launch_bounds__(256, 1) void tile_kernel(Product a, int base) {
    extern __shared__ __attribute__((aligned(1024))) uint8_t ring[];
    // Workgroups go to the 8 XCDs in turn: each XCD has a run of neighbouring tiles, BAND column tiles abreast, whose
    // rows and columns stay in its L2.
    const int blocks_m = (a.nrows + TM - 1) / TM;
    const int n_tiles = a.tiles ? *a.n_tiles : (a.ncols + TN - 1) / TN, total = n_tiles * blocks_m;
    const int xcd = blockIdx.x & 7, run = (total >> 3) + (xcd < (total & 7));
    // What is left of an XCD's run after whole rounds of its CUs, if at most half of one, goes in half tiles: half of
    // them among the first, so that the CUs store their results at different times.
    const int left = run % NEIGHBOURS, cut = HALVES && left <= NEIGHBOURS / 2 ? left : 0, full = run - cut;
    const int ahead = min(full, NEIGHBOURS / 2);
    const int turn = base + (blockIdx.x >> 3);
    if (turn >= full + 2 * cut) return;
    int at = turn, half = -1;
    if (turn >= ahead && turn < ahead + cut)
        half = turn - ahead;
    else if (turn >= full + cut)
        half = turn - full;
    else if (turn >= ahead)
        at = turn - cut;
    if (half >= 0) at = full + (half >> 1);
    const int id = xcd * (total >> 3) + min(xcd, total & 7) + at;
    int first, end, m0;
    const int8_t *w = a.w;
    const float *w_scale = a.w_scale;
    if (a.tiles) {
        const int t = id / blocks_m;
        const int4 spec = reinterpret_cast<const int4 *>(a.tiles)[t];
        w += spec.x * a.expert_stride;
        w_scale += (int64_t)spec.x * a.nrows;
        first = spec.y;
        end = spec.z;
        m0 = (id - t * blocks_m) * TM;
    } else {
        constexpr int BAND = 4;
        const int band = id / (BAND * blocks_m), in = id - band * BAND * blocks_m;
        const int wide = min(BAND, n_tiles - band * BAND);
        first = (band * BAND + in % wide) * TN;
        end = min(first + TN, a.ncols);
        m0 = in / wide * TM;
    }
    if constexpr (HALVES) {
        // Half of a tile's columns; a tile with no more than that is done by its first half.
        if (half >= 0 || end - first <= TN / 2) {
            if (half >= 0 && half & 1) first += TN / 2;
            if (half >= 0 && !(half & 1)) end = min(end, first + TN / 2);
            if (first < end) tile<TM, TN / 2, 3, 3, 1>(a, ring, w, w_scale, m0, first, end);
            return;
        }
    }
    tile<TM, TN, SW, SX, G>(a, ring, w, w_scale, m0, first, end);
}

template <int TM, int TN, int SW, int SX, int G, bool HALVES = false>
int launch(const Product &p, int64_t max_tiles, hipStream_t s) {
    int64_t total = max_tiles * ((p.nrows + TM - 1) / TM);
    total = (total + 7) / 8;
    if (HALVES) total += std::min(total, (int64_t)NEIGHBOURS / 2);
    constexpr int bytes = std::max((TM * SW + TN * SX) * STAGE, TM / 8 * 2048 + (TM + 2 * TN + 4) * 4);
    constexpr int64_t MOST = 1 << 18;  // of an XCD in one launch
    for (int64_t base = 0; base < total; base += MOST) {
        hipLaunchKernelGGL((tile_kernel<TM, TN, SW, SX, G, HALVES>), dim3((unsigned)std::min(total - base, MOST) * 8),
                           dim3(256), bytes, s, p, (int)base);
        if (const int e = (int)hipGetLastError()) return e;
    }
    return 0;
}

}  // namespace

// The largest tile of which there are enough: by the time of a stage and of a tile's start and end, a large one on some
// CUs beats small ones on all of them early.  Measured, us:
//   14336 x 4096 by 512: 112 of 256 x 256 39, 448 of 128 x 128 42, two a CU; by 128: 224 of 128 x 64 22.9, 448 of 64 x 64 23.5
//   4096 x 4096 by 1536: 96 of 256 x 256 36.9, 384 of 128 x 128 35.3; by 1024: 64 of 256 x 256 34.8, 256 of 128 x 128 23.9
//     with four stages, one a CU, 29.1 with two; by 512: 128 of 128 x 128 19.6, 256 of 128 x 64 19.1; by 256: 128 of
//     128 x 64 17.0, 256 of 64 x 64 12.6
//   5003 x 2720 by 333: 120 of 128 x 128 16.8, 240 of 128 x 64 14.8, 474 of 64 x 64 16.5
TileForm i8::tile_form(int64_t nrows, int64_t ncols) {
    auto tiles = [&](int64_t m, int64_t n) { return ((nrows + m - 1) / m) * ((ncols + n - 1) / n); };
    if (tiles(256, 256) >= 100) return TILE_256x256;
    if (tiles(128, 128) > 256) return TILE_128x128;
    if (tiles(128, 128) >= 140) return TILE_128x128_DEEP;
    if (tiles(128, 64) >= 200) return TILE_128x64;
    return TILE_64x64;
}

// (256 x 128, two a CU: 8192 x 768 by 8192 89 for 97 in 256 x 256, 8192 x 1200 153 for 133, 33880 pairs by 44 experts of
// 1039 x 723 13 us more than 128 x 128: not taken.)
//
// By experts, whose last tiles are half full on the average.  The smallest where there are few tiles, as above; tall narrow
// ones for experts with few columns; else 256 x 256 if rounds of them and their start and end, 15 us a tile, are few beside
// the work.  Measured (weight rows x inner, pairs by experts), us:
//   282 x 842, 1360 by 8: 6.0 in 64 x 64, 7.9 in 128 x 64, 9.6 in 128 x 128, 15.8 in 256 x 256
//   2048 x 2048, 1024 by 8: 17.5, 15.7, 17.8, 21.2
//   1536 x 2048, 8192 by 128: 116, 108, 117, 111; 16384: 174, 145, 141, 131; 32768: -, -, 209, 194
//   2027 x 1209, 3921 by 23 (184 of 256 x 256): 34.1, 32.3, 29.9, 34.1;  1039 x 723, 33880 by 44: 98, 79, 64, 75
TileForm i8::tile_form_grouped(int64_t K, int64_t nrows, int64_t n_as, int64_t n_pairs) {
    const int64_t experts = std::min(n_pairs, n_as);
    auto tiles = [&](int64_t m, int64_t n) { return (nrows + m - 1) / m * (n_pairs / n + experts / 2); };
    if (tiles(128, 64) < 200) return TILE_64x64;
    if (n_pairs <= 64 * experts || tiles(128, 128) < 400) return TILE_128x64;
    return K >= 1024 && tiles(256, 256) >= 600 ? TILE_256x256 : TILE_128x128;
}

int i8::tile_columns(TileForm form) {
    return form == TILE_256x256 ? 256 : form == TILE_128x128 || form == TILE_128x128_DEEP ? 128 : 64;
}

int i8::tile_product(const Product &p, TileForm form, int64_t max_tiles, hipStream_t s) {
    switch (form) {
    case TILE_64x64: return launch<64, 64, 4, 4, 4>(p, max_tiles, s);
    case TILE_128x64: return launch<128, 64, 3, 3, 2>(p, max_tiles, s);
    case TILE_128x128: return launch<128, 128, 2, 2, 1>(p, max_tiles, s);
    case TILE_128x128_DEEP: return launch<128, 128, 4, 4, 2>(p, max_tiles, s);
    default: return launch<256, 256, 3, 2, 1, true>(p, max_tiles, s);
    }
}
