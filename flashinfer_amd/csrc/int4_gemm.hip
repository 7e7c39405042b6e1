// Which kernel takes a product with 4-bit weights (mi_layer_int4_matmul).
//
//   out[m, n] = sum_g scale[g, n] (sum_{k in g} x[m, k] q[n, k]) + bias[n]
#include <stdlib.h>

#include "int4_common.hpp"

namespace miexp {

// Rows of x that start at multiples of 16 bytes and end at one are read as they
// are; others are copied, in 16 bits, to such rows with zeros at their end.
bool int4_aligned(const mi_layer_int4_args& a) {
    return (uint64_t)a.x % 16 == 0 && a.x_stride % 8 == 0 && a.K % 8 == 0;
}

__global__ __launch_bounds__(256) void int4_copy_kernel(const uint16_t* __restrict__ x, int64_t stride, int64_t rows,
                                                        int K, int ld, uint16_t* __restrict__ to) {
    const int pieces = ld / 8;
    for (int64_t row = blockIdx.x; row < rows; row += gridDim.x)
        for (int i = threadIdx.x; i < pieces; i += 256) {
            v4u w = {0, 0, 0, 0};
#pragma unroll
            for (int v = 0; v < 8; ++v)
                if (i * 8 + v < K) w[v / 2] |= (uint32_t)x[row * stride + i * 8 + v] << (16 * (v & 1));
            *reinterpret_cast<v4u*>(to + row * ld + i * 8) = w;
        }
}

// Whether the 32-bit offsets of the tiled kernels reach all of a tile's rows
// (of x's, if they are gathered) and an expert's scales.
bool int4_offsets_fit(const Int4Call& p) {
    const int64_t most = ((int64_t)1 << 32) - 512;
    return (p.row_ids ? p.a_rows : (int64_t)256) * p.x_stride * 2 < most && p.scale_expert * 4 < most;
}

Int4Tile pick_tile(const Int4Call& p) {
    const int64_t groups = p.offsets ? p.E : 1, rows = (p.rows + groups - 1) / groups;
    if (rows <= 4 && !p.offsets) return Int4Tile::T4x16;
    if (rows <= 16) return p.offsets ? Int4Tile::T16x128 : Int4Tile::T16x16;
    if (rows <= 32) return Int4Tile::T32x64;
    if (rows <= 64) return Int4Tile::T64x128;
    auto tiles = [&](int bm, int bn) { return groups * ((rows + bm - 1) / bm) * ((p.N + bn - 1) / bn); };
    if (tiles(64, 128) <= 256) return Int4Tile::T64x128;
    if (tiles(128, 128) <= 256) return Int4Tile::T128x128;
    return Int4Tile::T256;
}

// Whether a launch of this tile holds fewer than 2^32 threads (of those of
// int4_row.hip, 4096 workgroups go over any number).
bool launch_fits(const Int4Call& p, Int4Tile tile) {
    static const struct { int bm, bn, threads; } form[] = {
        {16, 32, 512}, {16, 64, 512}, {16, 128, 512}, {32, 64, 512}, {32, 128, 512}, {64, 64, 512},
        {64, 128, 512}, {128, 64, 512}, {128, 128, 512}, {256, 128, 512}};
    if (tile <= Int4Tile::T16x16) return true;
    const auto& f = form[(int)tile - (int)Int4Tile::T16x32];
    return max_tiles(p.rows, f.bm, p.E) * ((p.N + f.bn - 1) / f.bn) * f.threads < (int64_t)1 << 32;
}

// MI_INT4_TILE = 0 .. 11 (an Int4Tile) takes that tile where a call can have it, for tests and timing.
Int4Tile forced_tile(const Int4Call& p, Int4Tile tile) {
    const char* env = getenv("MI_INT4_TILE");
    if (env && *env) {
        const int v = atoi(env);
        if (v >= 0 && v < (int)Int4Tile::END) tile = (Int4Tile)v;
    }
    return tile <= Int4Tile::T16x16 || (launch_fits(p, tile) && int4_offsets_fit(p)) ? tile : Int4Tile::T16x16;
}

hipError_t launch_int4_matmul(const mi_layer_int4_args& a, hipStream_t s) {
    Int4Call p;
    p.x = a.x;
    p.w = a.w;
    p.scale = a.scale;
    p.bias = a.bias;
    p.out = a.out;
    p.offsets = a.num_experts ? a.expert_offsets : nullptr;
    p.row_ids = a.row_ids;
    p.a_rows = a.x_rows;
    p.rows = a.rows;
    p.x_stride = a.x_stride;
    p.out_stride = a.out_stride;
    p.N = (int)a.N;
    p.K = (int)a.K;
    p.KT = (p.K + 127) / 128;
    p.Np = (p.N + 15) / 16 * 16;
    p.group_shift = 0;
    while (1 << p.group_shift < a.group_size) ++p.group_shift;
    p.w_expert = (int64_t)p.Np * 64 * p.KT;
    p.scale_expert = (int64_t)p.Np * ((a.K + a.group_size - 1) / a.group_size);
    p.E = a.num_experts;
    p.bias_dtype = a.bias_dtype;
    p.out_dtype = a.out_dtype;
    p.zero_rest = a.num_experts != 0 && a.zero_rest != 0;
    p.w_large = (p.E ? p.E : 1) * p.w_expert > ((int64_t)256 << 20);
    if (!int4_aligned(a)) {
        const int ld = (p.K + 7) / 8 * 8;
        hipLaunchKernelGGL(int4_copy_kernel, dim3((unsigned)(p.a_rows < MAX_BLOCKS ? p.a_rows : MAX_BLOCKS)), dim3(256),
                           0, s, (const uint16_t*)p.x, p.x_stride, p.a_rows, p.K, ld, (uint16_t*)a.workspace);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
        p.x = a.workspace;
        p.x_stride = ld;
        p.K = ld;  // zeros past K
    }
    const uint64_t quad = a.out_dtype == MI_LAYER_F32 ? 16 : 8;
    const bool vec = (uint64_t)a.out % quad == 0 && a.out_stride % 4 == 0;
    const Int4Tile tile = forced_tile(p, pick_tile(p));
    if (tile <= Int4Tile::T16x16) return launch_int4_row(p, a.x_dtype, a.scale_dtype, tile, vec, s);
    if (tile == Int4Tile::T256) return launch_int4_wide(p, a.x_dtype, a.scale_dtype, vec, s);
    return launch_int4_tile(p, a.x_dtype, a.scale_dtype, tile, vec, s);
}

}  // namespace miexp
