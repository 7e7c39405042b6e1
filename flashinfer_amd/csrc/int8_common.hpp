// Shared by the integer product kernels: the arguments of a launch and the epilogue.
#pragma once

#include "grouped.hpp"
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

// Kernels for any operands, and for those whose strides and addresses are
// multiples of 16.
bool int8_offsets_fit(const Int8Call& p, int bm, int bn);  // a tile's lane offsets within 32 bits
enum class Int8Tile { T32x32, T32x64, T64x64_K2, T64x64, T64x128_K2, T64x128, T128x128_K2, T128x128, T256x256 };
hipError_t launch_pack_rows(const Int8Call& p, int8_t* to, int ld, hipStream_t s);
hipError_t launch_int8_any(const Int8Call& p, int out_dtype, Int8Tile tile, bool vec, hipStream_t s);
hipError_t launch_int8_tile(const Int8Call& p, int out_dtype, Int8Tile tile, bool vec, hipStream_t s);
hipError_t launch_int8_wide(const Int8Call& p, int out_dtype, hipStream_t s);

}  // namespace miexp
