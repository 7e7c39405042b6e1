// Which kernel takes a product of 8-bit integers (mi_experts_int8_matmul).
//
//   out[m, n] = (sum_k a[m, k] b[n, k]) a_scale[m] b_scale[n] + bias[n]
//
// The sum is exact in int32 (K <= 131071), so neither the order of k nor a
// split of it changes a result: all kernels agree bit for bit.
#include <stdlib.h>

#include "int8_common.hpp"

namespace miexp {

// A lane's offset: that of its row and a chunk inside 128 bytes. (Rows may
// overlap, so the chunk is not inside the row's own distance.)
bool int8_offsets_fit(const Int8Call& p, int bm, int bn) {
    const int64_t most = ((int64_t)1 << 32) - 128;
    return (p.row_ids ? p.a_rows : (int64_t)bm) * p.a_stride < most && bn * p.b_stride < most;
}

// The tile of a product. Tiles are taken as large as still give each CU one
// (256 of them), and K is shared inside a workgroup where that is what is left
// to share. Experts with more tiles than that take tiles that hold their rows,
// so that their weights are read once: those are what bounds the call. wide:
// 256 x 256 tiles are there too.
// The rows of an expert are known on the device alone. The host takes the rows
// of the result over all experts, which a shard fills in part: with 32 of 256
// experts it takes tiles for eight times the rows (4096 x 7168, 8 slots a token,
// by the rule and by the best tile: 400 tokens 192 / 144 us with 64 x 128, 1000
// 199 / 154 with 64 x 128, 3000 216 / 186 with 128 x 128, 8192 310 / 302 with the
// rule's; 64 125 / 124). Experts that cannot have a row count as well: 2 rows 28 /
// 16 with 32 x 32, but 8 rows of one token 37 / 37.
Int8Tile pick_tile(const Int8Call& p, bool wide) {
    const int64_t groups = p.offsets ? p.E : 1, rows = (p.rows + groups - 1) / groups;
    auto tiles = [&](int bm, int bn) { return groups * ((rows + bm - 1) / bm) * ((p.N + bn - 1) / bn); };
    if (tiles(32, 32) <= 256) return Int8Tile::T32x32;
    if (tiles(32, 64) <= 256) return Int8Tile::T32x64;
    if (tiles(64, 64) <= 256) return Int8Tile::T64x64_K2;
    // 48 KB of LDS: three to a CU (M = 700, N = 4096: K = 2048 12.9 against 15.5
    // us with 128 x 128 and K shared, K = 4096 24.2 against 23.6)
    if (tiles(64, 64) <= 768 && p.K <= 2048) return Int8Tile::T64x64;
    if (tiles(64, 128) <= 256) return Int8Tile::T64x128_K2;
    if (p.offsets && rows <= 40) return Int8Tile::T64x128;
    if (tiles(128, 128) <= 256) return Int8Tile::T128x128_K2;
    if (tiles(128, 128) <= 512 || !wide || (p.offsets && rows <= 96)) return Int8Tile::T128x128;
    // A second round of 256 x 256 tiles that leaves most CUs idle: smaller ones,
    // two to a CU, end more evenly (N = 4096, K = 7168: M = 4330 139 against 156
    // us, 5120 152 / 160, 6144 182 / 164; M = 2200, one round, 88 / 80).
    const int64_t rounds = (tiles(256, 256) + 255) / 256;
    if (!p.offsets && rounds > 1 && tiles(128, 128) * 3 < rounds * 2048) return Int8Tile::T128x128;
    return Int8Tile::T256x256;
}

// Whether a launch of this tile (forms as in launch_int8_tile; of the 256 x 256
// ones at most 256 workgroups run) holds fewer than 2^32 threads. Calls are
// bounded by their 64 x 64 tiles, which is enough for what pick_tile takes:
// smaller ones only for a few hundred.
bool launch_fits(const Int8Call& p, Int8Tile tile) {
    static const struct { int bm, bn, threads; } form[] = {
        {32, 32, 1024}, {32, 64, 1024}, {64, 64, 512}, {64, 64, 256}, {64, 128, 512}, {64, 128, 256},
        {128, 128, 512}, {128, 128, 256}};
    if (tile == Int8Tile::T256x256) return true;
    const auto& f = form[(int)tile];
    return max_tiles(p.rows, f.bm, p.E) * ((p.N + f.bn - 1) / f.bn) * f.threads < (int64_t)1 << 32;
}

// MI_INT8_TILE = 0 .. 8 (an Int8Tile) takes that tile where a call can have it, for tests and timing.
Int8Tile forced_tile(const Int8Call& p, bool wide, Int8Tile tile) {
    const char* env = getenv("MI_INT8_TILE");
    if (!env || !*env) return tile;
    const int v = atoi(env);
    if (v < 0 || v > (int)Int8Tile::T256x256 - !wide) return tile;
    return launch_fits(p, (Int8Tile)v) ? (Int8Tile)v : tile;
}

// Dense products whose K is no multiple of 16 are copied to rows that are one
// where that is less than what the kernels for any address lose: from 2^20 tiles
// x bytes of K on (8192 x 4096 x 7169 414 -> 227 to 237 us, 2048 x 4096 x 7169
// 127 -> 110, 3000 x 4000 x 1030 level, 1500 x 4096 x 2050 33.9 against 35.4).
// Strides and addresses do not count: the size of the workspace goes by the
// sizes alone. Bytes of the copies, 0 for none.
size_t int8_workspace(int64_t rows, int64_t N, int64_t K, int E) {
    const int64_t tiles = (rows + 127) / 128 * ((N + 127) / 128);
    const int64_t bytes = (rows + N) * ((K + 15) / 16 * 16);
    const bool copy = E == 0 && K % 16 != 0 && tiles > 256 && tiles * K > 1 << 20;
    return copy && bytes <= (int64_t)1 << 30 ? (size_t)bytes : 0;
}

hipError_t launch_int8_matmul(const mi_experts_int8_args& a, hipStream_t s) {
    Int8Call p;
    p.a = a.a;
    p.a_scale = a.a_scale;
    p.b = a.b;
    p.b_scale = a.b_scale;
    p.bias = a.bias;
    p.out = a.out;
    p.offsets = a.num_experts ? a.expert_offsets : nullptr;
    p.row_ids = a.row_ids;
    p.a_rows = a.a_rows;
    p.rows = a.rows;
    p.N = (int)a.N;
    p.K = (int)a.K;
    p.a_stride = a.a_stride;
    p.b_stride = a.b_stride;
    p.b_expert_stride = a.b_expert_stride;
    p.out_stride = a.out_stride;
    p.E = a.num_experts;
    p.bias_dtype = a.bias_dtype;
    p.zero_rest = a.num_experts != 0 && a.zero_rest != 0;
    p.b_large = (a.num_experts ? a.num_experts : 1) * a.N * a.K > ((int64_t)256 << 20);
    if (int8_workspace(a.rows, a.N, a.K, a.num_experts)) {
        const int ld = (p.K + 15) / 16 * 16;
        int8_t* to = (int8_t*)a.workspace;
        const hipError_t e = launch_pack_rows(p, to, ld, s);
        if (e != hipSuccess) return e;
        p.a = to;
        p.b = to + p.a_rows * ld;
        p.a_stride = p.b_stride = ld;
        p.K = ld;  // zeros past K
    }
    const uint64_t bits = (uint64_t)p.a | (uint64_t)p.b | (uint64_t)p.a_stride | (uint64_t)p.b_stride |
                          (uint64_t)p.b_expert_stride;
    const uint64_t quad = a.out_dtype == MI_EXPERTS_F32 ? 16 : 8;
    const bool vec = (uint64_t)a.out % quad == 0 && a.out_stride % 4 == 0;
    const bool fast = bits % 16 == 0 && p.K % 16 == 0 && int8_offsets_fit(p, 256, 256);
    const bool wide = fast && p.K > 128;  // the 256 x 256 kernel takes two steps of 128 bytes at least
    const Int8Tile tile = forced_tile(p, wide, pick_tile(p, wide));
    if (tile == Int8Tile::T256x256) return launch_int8_wide(p, a.out_dtype, s);
    if (fast) return launch_int8_tile(p, a.out_dtype, tile, vec, s);
    return launch_int8_any(p, a.out_dtype, tile, vec, s);
}

}  // namespace miexp
