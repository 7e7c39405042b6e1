// Shared by the products with 4-bit weights: the arguments of a launch, weights
// to 16 bits, and the epilogue.
#pragma once

#include "grouped.hpp"
#include "layer_common.hpp"

namespace miexp {

typedef unsigned v4u __attribute__((ext_vector_type(4)));
typedef float v4f __attribute__((ext_vector_type(4)));

// Device-side arguments of one product (see mi_layer_int4_args).
struct Int4Call {
    const void* x;
    const uint8_t* w;
    const void* scale;
    const void* bias;
    void* out;
    const int32_t* offsets;  // null: dense
    const int32_t* row_ids;  // null: row m of x
    int64_t a_rows, rows;    // a_rows: of x
    int64_t x_stride, out_stride;
    int64_t w_expert, scale_expert;  // bytes of an expert's weights, elements of its scales
    int N, K;
    int KT;           // tiles of 128 values: ceil(K / 128)
    int Np;           // channels of a row of scales
    int group_shift;  // log2 of the group size
    int E;
    int bias_dtype, out_dtype;
    int zero_rest;
    int64_t from_rows, to_rows;  // a launch that finds another number of rows with experts does nothing
};

// Whether this launch is the one for the rows that experts have.
__device__ __forceinline__ bool is_for_rows(const Int4Call& p) {
    if (!p.offsets || (p.from_rows == 0 && p.to_rows > p.rows)) return true;
    const int64_t n = clamped(p.offsets, p.E, p.rows) - clamped(p.offsets, 0, p.rows);
    return n >= p.from_rows && n < p.to_rows;
}

// Element types of x: its fragments, its matrix instruction, and the eight
// weights of a word.
//
// v_mfma_f32_16x16x32: lane l gives 8 values of row l % 16 of each operand (k =
// 8 * (l / 16) ..), and holds D[4 * (l / 16) + i][l % 16], i = 0..3, with rows
// of D from the first operand. Weights are the first operand everywhere here: a
// lane then holds four neighbouring output channels of one row.
//
// Integers of 4 bits are exact in both types, so a weight is rounded nowhere:
// sums of a group are products of x and whole numbers, and the scale is applied
// to the sums, in fp32.
template <class XT> struct Operand;

// v_cvt_off_f32_i4 makes q / 16 of the low 4 bits in two's complement, and the
// upper half of that is it in bfloat16: 13 instructions for eight values, as it
// can take its bits from any byte. As a builtin, not in assembly: behind a matrix
// instruction that still reads its addend from the registers that a vector
// instruction writes there have to be wait states, which the compiler counts for
// its own instructions alone.
template <> struct Operand<__bf16> {
    typedef __bf16 frag __attribute__((ext_vector_type(8)));
    static constexpr float UNIT = 16.f;  // weights are made as sixteenths, and sums are multiplied at their end
    __device__ __forceinline__ static frag weights(uint32_t d) {
        uint32_t h = d >> 4;
        asm("" : "+v"(h));  // bytes of this word, not bit fields of d: they cost an instruction less
        float e[8];  // nibbles 0 .. 7
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            e[2 * i] = __builtin_amdgcn_cvt_off_f32_i4((int)(d >> 8 * i & 0xffu));
            e[2 * i + 1] = __builtin_amdgcn_cvt_off_f32_i4((int)(h >> 8 * i & 0xffu));
        }
        v4u r;
#pragma unroll
        for (int i = 0; i < 4; ++i)
            r[i] = __builtin_amdgcn_perm(__float_as_uint(e[i + 4]), __float_as_uint(e[i]), 0x07060302u);
        return __builtin_bit_cast(frag, r);
    }
    __device__ __forceinline__ static v4f mfma(frag w, frag x, v4f c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(w, x, c, 0, 0, 0);
    }
};

// The bits of q + 8 as the last ones of 1024 (or, 4 bits up, as sixteenths of
// it), and 1032 off again: 9 instructions for eight values. The way of Kim,
// Henry, Fahim, Awadalla: Who says elephants can't run: bringing large scale MoE
// models into cloud scale production (2022); the numbers follow from the format.
template <> struct Operand<_Float16> {
    typedef _Float16 frag __attribute__((ext_vector_type(8)));
    static constexpr float UNIT = 1.f;
    __device__ __forceinline__ static frag weights(uint32_t d) {
        typedef _Float16 h2 __attribute__((ext_vector_type(2)));
        const uint32_t u = d >> 8;
        const h2 low = {(_Float16)1032.f, (_Float16)1032.f}, high = {(_Float16)72.f, (_Float16)72.f};
        const h2 part = {(_Float16)0.0625f, (_Float16)0.0625f};
        const h2 a = __builtin_bit_cast(h2, (d & 0x000f000fu) ^ 0x64086408u);
        const h2 b = __builtin_bit_cast(h2, (d & 0x00f000f0u) ^ 0x64806480u);
        const h2 c = __builtin_bit_cast(h2, (u & 0x000f000fu) ^ 0x64086408u);
        const h2 e = __builtin_bit_cast(h2, (u & 0x00f000f0u) ^ 0x64806480u);
        const h2 r[4] = {a - low, b * part - high, c - low, e * part - high};
        return frag{r[0][0], r[0][1], r[1][0], r[1][1], r[2][0], r[2][1], r[3][0], r[3][1]};
    }
    __device__ __forceinline__ static v4f mfma(frag w, frag x, v4f c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(w, x, c, 0, 0, 0);
    }
};

__device__ __forceinline__ float bias_at(const Int4Call& p, int n) {
    if (!p.bias) return 0.f;
    if (p.bias_dtype == MI_LAYER_F32) return reinterpret_cast<const float*>(p.bias)[n];
    if (p.bias_dtype == MI_LAYER_BF16) return (float)reinterpret_cast<const __bf16*>(p.bias)[n];
    return (float)reinterpret_cast<const _Float16*>(p.bias)[n];
}

template <class T>
__device__ __forceinline__ void store_channels(const Int4Call& p, int64_t m, int n, bool vec, const float (&y)[4]) {
    T* to = reinterpret_cast<T*>(p.out) + m * p.out_stride + n;
    if (vec && n + 4 <= p.N) {
        store<T, 4>(to, y);
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (n + i < p.N) to[i] = (T)y[i];
    }
}

// Results of channels n .. n + 3 of row m from their sums, which are in units of
// Op's weights; NaN for a row that is none of x.
template <class Op>
__device__ __forceinline__ void finish_sums(const Int4Call& p, int64_t m, int n, v4f sum, float (&y)[4]) {
    const bool none = source_row(p, m) < 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        y[i] = sum[i] * Op::UNIT;
        if (p.bias) y[i] += bias_at(p, min(n + i, p.N - 1));
        if (none) y[i] = __builtin_nanf("");
    }
}

template <class Op>
__device__ __forceinline__ void store_sums(const Int4Call& p, int64_t m, int n, bool vec, v4f sum) {
    if (n >= p.N) return;
    float y[4];
    finish_sums<Op>(p, m, n, sum, y);
    if (p.out_dtype == MI_LAYER_F32)
        store_channels<float>(p, m, n, vec, y);
    else if (p.out_dtype == MI_LAYER_F16)
        store_channels<_Float16>(p, m, n, vec, y);
    else
        store_channels<__bf16>(p, m, n, vec, y);
}

__device__ __forceinline__ void zero_rest_any(const Int4Call& p, bool vec) {
    if (p.out_dtype == MI_LAYER_F32)
        zero_rest<float>(p, vec);
    else if (p.out_dtype == MI_LAYER_F16)
        zero_rest<_Float16>(p, vec);
    else
        zero_rest<__bf16>(p, vec);
}

// Calls f(XT{}, ST{}, IntC<steps of 32 values that a scale holds for inside 128>).
template <class F>
hipError_t by_int4_types(int x_dtype, int scale_dtype, int group, F f) {
    auto steps = [&](auto x, auto s) {
        if (group == 32) return f(x, s, IntC<1>{});
        if (group == 64) return f(x, s, IntC<2>{});
        return f(x, s, IntC<4>{});
    };
    if (x_dtype == MI_LAYER_F16)
        return scale_dtype == MI_LAYER_F32 ? steps(_Float16{}, float{}) : steps(_Float16{}, _Float16{});
    return scale_dtype == MI_LAYER_F32 ? steps(__bf16{}, float{}) : steps(__bf16{}, __bf16{});
}

// Rows x channels of a workgroup. T4x16 and T16x16 are those of int4_row.hip,
// T256 that of int4_wide.hip.
enum class Int4Tile { T4x16, T16x16, T16x32, T16x64, T16x128, T32x64, T32x128, T64x64, T64x128, T128x128, T256, END };
hipError_t launch_int4_tile(const Int4Call& p, int x_dtype, int scale_dtype, Int4Tile tile, bool vec, hipStream_t s);
hipError_t launch_int4_wide(const Int4Call& p, int x_dtype, int scale_dtype, hipStream_t s);
hipError_t launch_int4_row(const Int4Call& p, int x_dtype, int scale_dtype, Int4Tile tile, bool vec, hipStream_t s);

}  // namespace miexp
