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

// Tiles of a dense product: the smallest that leave at most one workgroup for
// each of the 256 CUs. What a call of few tiles waits for is the chain of one
// workgroup's steps, and small tiles have more groups of waves that share K
// (4096 x 7168: 1 row 7.7 us, 16 8.8, 32 11.5, with 16 x 64 tiles 17; 64 rows
// 17.4, with 16 x 32 20.6; 100 20.2 / 23.7 with 16 x 64; 256 26 / 27.6 with 32 x
// 64; 512 41 / 52 with 64 x 64; 1024 74 / 80 with 64 x 128).
// Where 64 x 64 tiles do not fit, two workgroups of a smaller one to a CU do better
// than one of 64 x 128, whatever K is (in groups of 128; 2048 / 7168 values of K; 160
// rows x 6144: 11.4 / 28.2 us with 480 tiles of 32 x 64, 13.6 / 36.5 with 480 of 16 x
// 128, 15.2 / 38.6 with 64 x 128; 144 x 7168: 16.0 / 41.6 with 560 of 32 x 64, 13.7 /
// 36.2 with 504 of 16 x 128, 15.2 / 38.7; 210 x 4700: 16.4 / 41.6 with 518 of 32 x 64,
// 20.0 / 55.7 with 518 of 16 x 128, 15.6 / 38.8); where they fit, one of those does
// (256 x 4096: 10.7 / 26.0, 13.5 / 35.5 with 512 of 16 x 128).
Int4Tile pick_dense(const Int4Call& p) {
    auto tiles = [&](int bm, int bn) { return ((p.rows + bm - 1) / bm) * ((p.N + bn - 1) / bn); };
    if (p.rows <= 4 && tiles(4, 16) <= 512) return Int4Tile::T4x16;
    if (tiles(16, 16) <= 256) return Int4Tile::T16x16;
    if (tiles(16, 32) <= 256) return Int4Tile::T16x32;
    if (tiles(16, 64) <= 256) return Int4Tile::T16x64;
    if (tiles(32, 64) <= 256) return Int4Tile::T32x64;
    if (tiles(64, 64) <= 256) return Int4Tile::T64x64;
    if (tiles(32, 64) <= 512) return Int4Tile::T32x64;
    if (tiles(16, 128) <= 512) return Int4Tile::T16x128;
    if (tiles(64, 128) <= 256) return Int4Tile::T64x128;
    if (tiles(128, 128) <= 256) return Int4Tile::T128x128;
    // A round of 256 x 192 tiles takes as long as three and a half of 64 x 128 ones
    // (4096 x 7168: 1500 rows, three rounds, 115 us / 134 with 256 x 192, 1750, four, 152 /
    // 135; 2048 x 1024: 2600 rows, three, 29.8 / 30.9, 3500, four, 38.9 / 30.5), one of 256
    // x 128 in smaller groups less than three (groups of 64, 1100 rows of 4096 x 7168, 114 /
    // 98, 1500 117 / 111, 2200 of 2048 x 1024 30 / 24).
    return p.group_shift >= 7 && tiles(64, 128) <= 3 * 256 ? Int4Tile::T64x128 : Int4Tile::T256;
}

// Rows of an expert on average up to which 32 x 128 tiles are taken, not those of
// 256 rows (32 experts with a router's spread; 4096 x 7168 in groups of 128: 56
// rows 194 us / 274, 80 271 / 277, 88 295 / 280, 112 349 / 304; in groups of 32 56
// rows 226 / 326, 80 300 / 340, 112 399 / 386; 7168 x 2048 56 rows 116 / 151, 80 151 /
// 160, 96 179 / 164).
constexpr int SMALL_ROWS = 80;

// Tiles of experts' products. The host knows the rows of the result, of which a
// shard's experts have a part (an eighth, if they are 32 of 256). Where that
// decides, both kernels are launched and one finds that the rows are not its own.
Int4Tile pick_grouped(const Int4Call& p, Int4Tile& large) {
    const int64_t rows = (p.rows + p.E - 1) / p.E;
    large = Int4Tile::END;
    // 16 x 128 reads the weights at the rate of memory (64 tokens, 8 of 256 experts
    // each, 32 of them here: 87 us for 425 MB)
    if (rows <= 32) return Int4Tile::T16x128;
    if (rows > 512) return Int4Tile::T256;
    if (rows > SMALL_ROWS) large = Int4Tile::T256;
    return Int4Tile::T32x128;
}

// Whether a launch of this tile holds fewer than 2^32 threads (of those of
// int4_row.hip, 4096 workgroups go over any number).
bool launch_fits(const Int4Call& p, Int4Tile tile) {
    static const struct { int bm, bn; } form[] = {{16, 32}, {16, 64}, {16, 128}, {32, 64}, {32, 128}, {64, 64},
                                                  {64, 128}, {128, 128}, {256, 128}};
    const auto& f = form[(int)tile - (int)Int4Tile::T16x32];
    return max_tiles(p.rows, f.bm, p.E) * ((p.N + f.bn - 1) / f.bn) * 512 < (int64_t)1 << 32;
}

hipError_t launch_one(const Int4Call& p, const mi_layer_int4_args& a, Int4Tile tile, hipStream_t s) {
    const uint64_t quad = a.out_dtype == MI_LAYER_F32 ? 16 : 8;
    const bool vec = (uint64_t)a.out % quad == 0 && a.out_stride % 4 == 0;
    if (tile > Int4Tile::T16x16 && !(launch_fits(p, tile) && int4_offsets_fit(p))) tile = Int4Tile::T16x16;
    if (tile <= Int4Tile::T16x16) return launch_int4_row(p, a.x_dtype, a.scale_dtype, tile, vec, s);
    if (tile == Int4Tile::T256) return launch_int4_wide(p, a.x_dtype, a.scale_dtype, s);
    return launch_int4_tile(p, a.x_dtype, a.scale_dtype, tile, vec, s);
}

// MI_INT4_TILE = 0 .. 10 (an Int4Tile) takes that tile where a call can have it, for tests and timing.
Int4Tile forced_tile() {
    const char* env = getenv("MI_INT4_TILE");
    const int v = env && *env ? atoi(env) : -1;
    return v >= 0 && v < (int)Int4Tile::END ? (Int4Tile)v : Int4Tile::END;
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
    p.from_rows = 0;
    p.to_rows = INT64_MAX;
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
    const Int4Tile forced = forced_tile();
    if (forced != Int4Tile::END) return launch_one(p, a, forced, s);
    if (!p.offsets) return launch_one(p, a, pick_dense(p), s);
    Int4Tile large;
    const Int4Tile tile = pick_grouped(p, large);
    // a tile that does not fit is one kernel for all
    if (large == Int4Tile::END || !int4_offsets_fit(p) || !launch_fits(p, tile)) return launch_one(p, a, tile, s);
    p.to_rows = SMALL_ROWS * p.E;
    const hipError_t e = launch_one(p, a, tile, s);
    if (e != hipSuccess) return e;
    p.from_rows = p.to_rows;
    p.to_rows = INT64_MAX;
    return launch_one(p, a, large, s);
}

}  // namespace miexp
