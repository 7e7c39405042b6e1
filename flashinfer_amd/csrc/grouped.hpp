// Shared by the products of rows with their experts' weights: which rows and
// expert a tile has. A call's arguments (Call) hold offsets (null: dense),
// row_ids (null: row m of a), a_rows, rows, E, N, out, out_stride, zero_rest.
#pragma once

#include "experts_common.hpp"

namespace miexp {

__device__ __forceinline__ int64_t clamped(const int32_t* offsets, int e, int64_t rows) {
    return max((int64_t)0, min((int64_t)offsets[e], rows));
}

// The experts' row tiles of BM rows, in order: ceil(rows / BM) of each. A wave
// looks at 64 experts at a time. Uniform over the workgroup.
struct Tiles {
    int e, first;   // expert, and its first row tile
    int tiles;      // its row tiles
    int row, end;   // its rows
};

// ceil(rows / BM) for up to 2^31 - 1 rows: BM - 1 more may have no place in 32 bits.
template <int BM>
constexpr int tiles_for(int rows) { return rows / BM + (rows % BM != 0); }
static_assert(tiles_for<16>(0) == 0 && tiles_for<16>(1) == 1 && tiles_for<16>(16) == 1 && tiles_for<16>(17) == 2 &&
                  tiles_for<4>(2147483647) == 536870912 && tiles_for<256>(2147483647) == 8388608,
              "a tile for every row");

// Row tiles of lane's expert e0 + lane (none past the last), and their inclusive sum.
template <int BM, class Call>
__device__ __forceinline__ int scan_tiles(const Call& p, int e0, int& lo, int& hi, int& inc) {
    const int lane = threadIdx.x & 63, x = e0 + lane;
    lo = hi = 0;
    if (x < p.E) {
        lo = (int)clamped(p.offsets, x, p.rows);
        hi = max(lo, (int)clamped(p.offsets, x + 1, p.rows));
    }
    const int tiles = tiles_for<BM>(hi - lo);
    inc = tiles;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const int u = __shfl_up(inc, d);
        if (lane >= d) inc += u;
    }
    return tiles;
}

// The expert that has row tile mt. False past the last tile.
template <int BM, class Call>
__device__ __forceinline__ bool find_expert(const Call& p, int mt, Tiles& t) {
    if (!p.offsets) {
        t = Tiles{0, 0, (int)((p.rows + BM - 1) / BM), 0, (int)p.rows};
        return mt < t.tiles;
    }
    int before = 0;
    for (int e0 = 0; e0 < p.E; e0 += 64) {
        int lo, hi, inc;
        const int tiles = scan_tiles<BM>(p, e0, lo, hi, inc);
        const unsigned long long has = __ballot(before + inc > mt);
        if (has) {
            const int l = __ffsll(has) - 1;
            t.e = __builtin_amdgcn_readfirstlane(e0 + l);
            t.first = __builtin_amdgcn_readfirstlane(before + __shfl(inc - tiles, l));
            t.tiles = __builtin_amdgcn_readfirstlane(__shfl(tiles, l));
            t.row = __builtin_amdgcn_readfirstlane(__shfl(lo, l));
            t.end = __builtin_amdgcn_readfirstlane(__shfl(hi, l));
            return true;
        }
        before += __builtin_amdgcn_readfirstlane(__shfl(inc, 63));
    }
    return false;
}

// Row tile mt: its expert, first row and rows.
template <int BM, class Call>
__device__ __forceinline__ bool find_tile(const Call& p, int mt, int& e, int64_t& row0, int& nrows) {
    Tiles t;
    if (!find_expert<BM>(p, mt, t)) return false;
    e = t.e;
    row0 = (int64_t)t.row + (int64_t)(mt - t.first) * BM;
    nrows = (int)min((int64_t)BM, t.end - row0);
    return true;
}

template <int BM, class Call>
__device__ __forceinline__ int count_tiles(const Call& p) {
    if (!p.offsets) return (int)((p.rows + BM - 1) / BM);
    int total = 0;
    for (int e0 = 0; e0 < p.E; e0 += 64) {
        int lo, hi, inc;
        scan_tiles<BM>(p, e0, lo, hi, inc);
        total += __builtin_amdgcn_readfirstlane(__shfl(inc, 63));
    }
    return total;
}

// Tile t of `total` in an order in which tiles that run at the same time share
// operands: an expert's row tiles go in groups of GM, channel tiles inside a
// group, row tiles innermost.
template <int BM, int GM, class Call>
__device__ __forceinline__ void tile_at(const Call& p, int t, int ntiles, int& e, int64_t& row0, int& nrows,
                                        int& nt) {
    Tiles x;
    find_expert<BM>(p, t / ntiles, x);
    const int u = t - x.first * ntiles;
    const int grp = u / (GM * ntiles), gm = min(GM, x.tiles - grp * GM), v = u - grp * GM * ntiles;
    nt = v / gm;
    e = x.e;
    row0 = (int64_t)x.row + (int64_t)(grp * GM + v - nt * gm) * BM;
    nrows = (int)min((int64_t)BM, x.end - row0);
}

// Row of a that feeds row m of the product; -1 for an id that is none.
template <class Call>
__device__ __forceinline__ int64_t source_row(const Call& p, int64_t m) {
    if (!p.row_ids) return m;
    const int64_t id = p.row_ids[m];
    return id >= 0 && id < p.a_rows ? id : -1;
}

// Zeros for the rows before the first expert's and behind the last one's, by
// all workgroups of a launch once their tiles are done (8192 rows, all in use,
// 256 for each of 32 experts of 7168 x 2048: 159 us with or without; a fill of
// the whole result before the product took 17 more). Rows that are not in use
// cost what writing them takes: 353 against 185 us where an eighth of 65536 is.
template <class T, class Call>
__device__ __forceinline__ void zero_rest(const Call& p, bool vec) {
    if (!p.zero_rest) return;
    const int64_t first = clamped(p.offsets, 0, p.rows), end = max(first, clamped(p.offsets, p.E, p.rows));
    for (int64_t i = blockIdx.x; i < first + p.rows - end; i += gridDim.x) {
        T* to = reinterpret_cast<T*>(p.out) + (i < first ? i : end + i - first) * p.out_stride;
        for (int n = threadIdx.x * 4; n < p.N; n += blockDim.x * 4) {
            const float zero[4] = {0.f, 0.f, 0.f, 0.f};
            if (vec && n + 4 <= p.N) {
                store<T, 4>(to + n, zero);
            } else {
                for (int v = n; v < min(n + 4, p.N); ++v) to[v] = (T)0.f;
            }
        }
    }
}

// Upper bound of row tiles: a tile each for the full ones, one more per expert.
inline int64_t max_tiles(int64_t rows, int bm, int E) {
    const int64_t full = (rows + bm - 1) / bm;
    return E ? (rows / bm + (rows < E ? rows : E)) : full;
}

// Calls f(T{}) with the float type of MI_EXPERTS_* dtype.
template <class F>
hipError_t by_out_type(int dtype, F f) {
    if (dtype == MI_EXPERTS_F32) return f(float{});
    if (dtype == MI_EXPERTS_F16) return f(_Float16{});
    return f(__bf16{});
}

}  // namespace miexp
