// Shared by the integer product kernels: the arguments of a launch, which rows
// and expert a tile has, and the epilogue.
#pragma once

#include "experts_common.hpp"
#include "lds_copy.hpp"

namespace miexp {

// Device-side arguments of one product (see mi_experts_int8_args).
struct Int8Call {
    const int8_t* a;
    const float* a_scale;
    const int8_t* b;
    const float* b_scale;
    const void* bias;
    void* out;
    const int32_t* offsets;  // null: dense
    const int32_t* row_ids;  // null: row m of a
    int64_t a_rows, rows;
    int N, K;
    int64_t a_stride, b_stride, b_expert_stride, out_stride;
    int E;
    int bias_dtype;
    int zero_rest;  // rows that no expert has get zeros
    int b_large;  // the weights exceed the 256 MB of the last cache
};

// v_mfma_i32_16x16x64_i8: lane l gives 16 bytes of row l % 16 of each operand
// (k = 16 * (l / 16) ..), and holds D[4 * (l / 16) + i][l % 16], i = 0..3, with
// rows of D from the first operand. Weights are the first operand everywhere
// here: a lane then holds four neighbouring output channels of one row.
__device__ __forceinline__ v4i mfma_i8(v4i w, v4i x, v4i c) {
    return __builtin_amdgcn_mfma_i32_16x16x64_i8(w, x, c, 0, 0, 0);
}

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

// Row tiles of lane's expert e0 + lane (none past the last), and their inclusive sum.
template <int BM>
__device__ __forceinline__ int scan_tiles(const Int8Call& p, int e0, int& lo, int& hi, int& inc) {
    const int lane = threadIdx.x & 63, x = e0 + lane;
    lo = hi = 0;
    if (x < p.E) {
        lo = (int)clamped(p.offsets, x, p.rows);
        hi = max(lo, (int)clamped(p.offsets, x + 1, p.rows));
    }
    const int tiles = (hi - lo + BM - 1) / BM;
    inc = tiles;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const int u = __shfl_up(inc, d);
        if (lane >= d) inc += u;
    }
    return tiles;
}

// The expert that has row tile mt. False past the last tile.
template <int BM>
__device__ __forceinline__ bool find_expert(const Int8Call& p, int mt, Tiles& t) {
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
template <int BM>
__device__ __forceinline__ bool find_tile(const Int8Call& p, int mt, int& e, int64_t& row0, int& nrows) {
    Tiles t;
    if (!find_expert<BM>(p, mt, t)) return false;
    e = t.e;
    row0 = (int64_t)t.row + (int64_t)(mt - t.first) * BM;
    nrows = (int)min((int64_t)BM, t.end - row0);
    return true;
}

template <int BM>
__device__ __forceinline__ int count_tiles(const Int8Call& p) {
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
template <int BM, int GM>
__device__ __forceinline__ void tile_at(const Int8Call& p, int t, int ntiles, int& e, int64_t& row0, int& nrows,
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
__device__ __forceinline__ int64_t source_row(const Int8Call& p, int64_t m) {
    if (!p.row_ids) return m;
    const int64_t id = p.row_ids[m];
    return id >= 0 && id < p.a_rows ? id : -1;
}

__device__ __forceinline__ float bias_at(const Int8Call& p, int n) {
    if (!p.bias) return 0.f;
    if (p.bias_dtype == MI_EXPERTS_F32) return reinterpret_cast<const float*>(p.bias)[n];
    if (p.bias_dtype == MI_EXPERTS_F16) return (float)reinterpret_cast<const _Float16*>(p.bias)[n];
    return (float)reinterpret_cast<const __bf16*>(p.bias)[n];
}

// 16 zero bytes: what copies past the end of K read.
static __device__ const v4i kZeros = {0, 0, 0, 0};
static __device__ const float kNan = __builtin_nanf("");  // the scale of a row that is none

__device__ __forceinline__ float row_scale(const Int8Call& p, int64_t row) {
    const int64_t from = source_row(p, row);
    return from >= 0 ? p.a_scale[from] : __builtin_nanf("");
}

// The scales and biases of a wave's MT x NT tiles: rows row_at + 16 m +
// lane % 16 of the tile, channels n_at + 16 n + 4 (lane / 16) .. Loaded before
// the products, used after them.
template <int MT, int NT>
struct Scales {
    float a[MT];
    float s[NT][4], b[NT][4];

    __device__ __forceinline__ void load(const Int8Call& p, int e, int64_t row0, int nrows, int row_at, int n_at) {
        const int lane = threadIdx.x & 63;
#pragma unroll
        for (int m = 0; m < MT; ++m) {
            const int row = row_at + m * 16 + (lane & 15);
            a[m] = row < nrows ? row_scale(p, row0 + row) : 0.f;
        }
        const float* scale = p.b_scale + (int64_t)e * p.N;
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int v = 0; v < 4; ++v) {
                s[n][v] = scale[min(n_at + n * 16 + 4 * (lane >> 4) + v, p.N - 1)];
                b[n][v] = 0.f;
            }
        if (p.bias) {
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int v = 0; v < 4; ++v) b[n][v] = bias_at(p, min(n_at + n * 16 + 4 * (lane >> 4) + v, p.N - 1));
        }
    }
};

// Stores a wave's tiles from their sums. vec: rows of out hold aligned groups
// of four.
template <class T, int MT, int NT>
__device__ __forceinline__ void store_tiles(const Int8Call& p, int64_t row0, int nrows, int row_at, int n_at, bool vec,
                                            const v4i (&acc)[MT][NT], const Scales<MT, NT>& c) {
    const int lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4;
    T* out = reinterpret_cast<T*>(p.out) + (row0 + row_at + r) * p.out_stride;
#pragma unroll
    for (int n = 0; n < NT; ++n) {
        const int at = n_at + n * 16 + 4 * g;
        if (at >= p.N) break;
#pragma unroll
        for (int m = 0; m < MT; ++m) {
            if (row_at + m * 16 + r >= nrows) continue;
            T* to = out + m * 16 * p.out_stride + at;
            float y[4];
#pragma unroll
            for (int v = 0; v < 4; ++v) y[v] = (float)acc[m][n][v] * c.a[m] * c.s[n][v] + c.b[n][v];
            if (vec && at + 4 <= p.N) {
                store<T, 4>(to, y);
            } else {
#pragma unroll
                for (int v = 0; v < 4; ++v)
                    if (at + v < p.N) to[v] = (T)y[v];
            }
        }
    }
}

// Zeros for the rows before the first expert's and behind the last one's, by
// all workgroups of a launch once their tiles are done (8192 rows, all in use,
// 256 for each of 32 experts of 7168 x 2048: 159 us with or without; a fill of
// the whole result before the product took 17 more). Rows that are not in use
// cost what writing them takes: 353 against 185 us where an eighth of 65536 is.
template <class T>
__device__ __forceinline__ void zero_rest(const Int8Call& p, bool vec) {
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

// Sums of the KS groups of four waves that shared K, in group 0. smem: the
// whole workgroup's, free once all are here.
template <int KS, int MT, int NT>
__device__ __forceinline__ void sum_groups(uint8_t* smem, int ks, int wave, v4i (&acc)[MT][NT]) {
    if constexpr (KS > 1) {
        __syncthreads();
        v4i* sum = reinterpret_cast<v4i*>(smem) + (wave * 64 + (threadIdx.x & 63));
        if (ks > 0) {
#pragma unroll
            for (int i = 0; i < MT * NT; ++i) sum[((ks - 1) * MT * NT + i) * 256] = acc[i / NT][i % NT];
        }
        __syncthreads();
        if (ks > 0) return;
#pragma unroll
        for (int i = 0; i < MT * NT; ++i)
#pragma unroll
            for (int k = 0; k < KS - 1; ++k) acc[i / NT][i % NT] += sum[(k * MT * NT + i) * 256];
    }
}

// Upper bound of row tiles: a tile each for the full ones, one more per expert.
inline int64_t max_tiles(int64_t rows, int bm, int E) {
    const int64_t full = (rows + bm - 1) / bm;
    return E ? (rows / bm + (rows < E ? rows : E)) : full;
}

// Kernels for any operands, and for those whose strides and addresses are
// multiples of 16.
bool int8_offsets_fit(const Int8Call& p, int bm, int bn);  // a tile's lane offsets within 32 bits
enum class Int8Tile { T32x32, T32x64, T64x64_K2, T64x64, T64x128_K2, T64x128, T128x128_K2, T128x128, T256x256 };
hipError_t launch_pack_rows(const Int8Call& p, int8_t* to, int ld, hipStream_t s);
hipError_t launch_int8_any(const Int8Call& p, int out_dtype, Int8Tile tile, bool vec, hipStream_t s);
hipError_t launch_int8_tile(const Int8Call& p, int out_dtype, Int8Tile tile, bool vec, hipStream_t s);
hipError_t launch_int8_wide(const Int8Call& p, int out_dtype, hipStream_t s);

// Calls f(T{}) with the float type of MI_EXPERTS_* dtype.
template <class F>
hipError_t by_out_type(int dtype, F f) {
    if (dtype == MI_EXPERTS_F32) return f(float{});
    if (dtype == MI_EXPERTS_F16) return f(_Float16{});
    return f(__bf16{});
}

}  // namespace miexp
