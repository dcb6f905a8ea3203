// i8_stream.hip -- the 8-bit product for few columns: weights go once from
// memory to registers, in the order the matrix instruction takes them.
//
// A workgroup takes 16 weight rows and up to 16 * NT columns; its waves deal
// the inner axis out in steps of 128 bytes.  Of a step lane (r, g) holds bytes
// 32 g .. 32 g + 31 of row r, as the operands of two 16x16x64 instructions: the
// order along the inner axis does not matter to a sum of integers as long as
// both operands have it.
#include <algorithm>

#include "i8.h"

using namespace i8;

namespace {

constexpr int WAVES = 8;
constexpr int STEP = 128;

template <int NT>
__global__ __launch_bounds__(64 * WAVES) void stream_kernel(Product a) {
    __shared__ v4i part[WAVES][NT][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r = lane & 15, g = lane >> 4;
    const int row_blocks = (a.nrows + 15) / 16, n_tiles = a.tiles ? *a.n_tiles : (a.ncols + 16 * NT - 1) / (16 * NT);
    for (int64_t b = blockIdx.x; b < (int64_t)row_blocks * n_tiles; b += gridDim.x) {
    const int tile = (int)(b / row_blocks), m0 = (int)(b - (int64_t)tile * row_blocks) * 16;
    int first = tile * 16 * NT, end = min(first + 16 * NT, a.ncols);
    const int8_t *w = a.w;
    const float *w_scale = a.w_scale;
    if (a.tiles) {
        const int4 t = reinterpret_cast<const int4 *>(a.tiles)[tile];
        w += t.x * a.expert_stride;
        w_scale += (int64_t)t.x * a.nrows;
        first = t.y;
        end = t.z;
    }
    w += (int64_t)min(m0 + r, a.nrows - 1) * a.w_stride;
    const int8_t *x[NT];
#pragma unroll
    for (int j = 0; j < NT; ++j) {
        const int c = min(first + 16 * j + r, end - 1);
        x[j] = a.x + (int64_t)(a.tiles ? a.col_src[c] : c) * a.x_stride;
    }
    v4i acc[NT];
#pragma unroll
    for (int j = 0; j < NT; ++j) acc[j] = (v4i){};
    const int whole = a.K / STEP;
    for (int step = wave; step < whole; step += WAVES) {
        const int k = step * STEP + g * 32;
#pragma unroll
        for (int h = 0; h < 32; h += 16) {
            const v4i u = *reinterpret_cast<const v4i *>(w + k + h);
#pragma unroll
            for (int j = 0; j < NT; ++j)
                acc[j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(u, *reinterpret_cast<const v4i *>(x[j] + k + h), acc[j], 0, 0, 0);
        }
    }
    if (whole * STEP < a.K && whole % WAVES == wave) {
#pragma unroll
        for (int h = 0; h < 32; h += 16) {
            const int k = whole * STEP + g * 32 + h;
            const bool any = k < a.K;  // chunks past K are not read
            v4i u = (v4i){};
            if (any) u = cut(*reinterpret_cast<const v4i *>(w + k), a.K - k);
#pragma unroll
            for (int j = 0; j < NT; ++j) {
                v4i v = (v4i){};
                if (any) v = *reinterpret_cast<const v4i *>(x[j] + k);
                acc[j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(u, v, acc[j], 0, 0, 0);
            }
        }
    }
#pragma unroll
    for (int j = 0; j < NT; ++j) part[wave][j][lane] = acc[j];
    __syncthreads();
    // Lane (r, g) of tile j has column r and rows 4 g .. 4 g + 3.
    for (int i = threadIdx.x; i < NT * 64; i += 64 * WAVES) {
        const int j = i >> 6, l = i & 63, c = first + 16 * j + (l & 15), m = m0 + 4 * (l >> 4);
        if (c >= end || m >= a.nrows) continue;
        v4i s = part[0][j][l];
#pragma unroll
        for (int q = 1; q < WAVES; ++q) s += part[q][j][l];
        const float xs = a.x_scale[a.tiles ? a.col_src[c] : c];
        float *out = a.dst + (int64_t)(a.tiles ? a.col_dst[c] : c) * a.dst_stride + m;
        for (int q = 0; q < min(4, a.nrows - m); ++q) out[q] = scaled(s[q], xs, w_scale[m + q]);
    }
    __syncthreads();
    }
}

}  // namespace

int i8::stream_product(const Product &p, int64_t max_tiles, int bn, hipStream_t s) {
    const dim3 grid((unsigned)std::min((p.nrows + 15) / 16 * max_tiles, (int64_t)1 << 20));
    const dim3 block(64 * WAVES);
    if (bn <= 16)
        hipLaunchKernelGGL(stream_kernel<1>, grid, block, 0, s, p);
    else if (bn <= 32)
        hipLaunchKernelGGL(stream_kernel<2>, grid, block, 0, s, p);
    else
        hipLaunchKernelGGL(stream_kernel<4>, grid, block, 0, s, p);
    return (int)hipGetLastError();
}
