// Shared by the integer product kernels: the arguments of a launch, which rows
// and expert a tile has, and the epilogue.
#pragma once

#include "experts_common.hpp"

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

// Row tile `mt` of BM rows: its expert, first row and rows. Experts have
// ceil(rows / BM) tiles each, in order; a wave looks at 64 of them at a time.
// False past the last tile. Uniform over the workgroup.
template <int BM>
__device__ __forceinline__ bool find_tile(const Int8Call& p, int64_t mt, int& e, int64_t& row0, int& nrows) {
    if (!p.offsets) {
        e = 0;
        row0 = mt * BM;
        if (row0 >= p.rows) return false;
        nrows = (int)min((int64_t)BM, p.rows - row0);
        return true;
    }
    const int lane = threadIdx.x & 63;
    int64_t before = 0;
    for (int e0 = 0; e0 < p.E; e0 += 64) {
        const int x = e0 + lane;
        int64_t lo = 0, hi = 0;
        if (x < p.E) {
            lo = clamped(p.offsets, x, p.rows);
            hi = max(lo, clamped(p.offsets, x + 1, p.rows));
        }
        const int tiles = (int)((hi - lo + BM - 1) / BM);
        int inc = tiles;
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            const int u = __shfl_up(inc, d);
            if (lane >= d) inc += u;
        }
        const unsigned long long has = __ballot(before + inc > mt);
        if (has) {
            const int l = __ffsll(has) - 1;
            e = __builtin_amdgcn_readfirstlane(e0 + l);
            const int at = __builtin_amdgcn_readfirstlane(__shfl(inc - tiles, l));
            const int first = __builtin_amdgcn_readfirstlane(__shfl((int)lo, l));
            const int end = __builtin_amdgcn_readfirstlane(__shfl((int)hi, l));
            row0 = first + (mt - before - at) * BM;
            nrows = (int)min((int64_t)BM, end - row0);
            return true;
        }
        before += __shfl(inc, 63);
    }
    return false;
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

// Upper bound of row tiles: a tile each for the full ones, one more per expert.
inline int64_t max_tiles(int64_t rows, int bm, int E) {
    const int64_t full = (rows + bm - 1) / bm;
    return E ? (rows / bm + (rows < E ? rows : E)) : full;
}

}  // namespace miexp
