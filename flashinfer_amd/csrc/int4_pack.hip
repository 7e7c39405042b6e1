// Weights of 4 bits laid out for their products (mi_layer_pack_int4), and made
// from floats with a scale for each group (mi_layer_quantize_int4). Once for
// each weight of a model, so simple: a thread makes a word of eight values.
// 32 x 4096 x 7168: packed in 470 us with its scales (1.41 GB read and written,
// 300 at the rate of a copy). From bfloat16 in groups of 128 2770 us, of 32 3200,
// from fp32 3480: the values are read twice, one at a time.
#include "int4_common.hpp"

namespace miexp {

// Where a word of the layout takes its values from: channel n, values k .. k + 7
// of expert e.
struct Int4Word {
    int64_t e, n, k;
};
__device__ __forceinline__ Int4Word int4_word(int64_t i, int64_t nt, int64_t kt) {
    const int in = (int)(i & 255), lane = in >> 2;
    const int64_t t = i >> 8, row = t / kt;
    return Int4Word{row / nt, (row % nt) * 16 + (lane & 15), (t - row * kt) * 128 + 32 * (in & 3) + 8 * (lane >> 4)};
}
// The even values in the low four nibbles, the odd ones in the high four.
__device__ __forceinline__ int int4_place(int v) { return 4 * ((v >> 1) + 4 * (v & 1)); }

// VEC: eight values are one load (32 x 4096 x 7168: 1720 us with a load each).
template <bool VEC>
__global__ __launch_bounds__(256) void pack_int4_kernel(const int8_t* __restrict__ q, int64_t expert_stride,
                                                        int64_t stride, int64_t words, int64_t N, int64_t K, int64_t nt,
                                                        int64_t kt, uint32_t* __restrict__ to) {
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < words; i += (int64_t)gridDim.x * 256) {
        const Int4Word a = int4_word(i, nt, kt);
        uint32_t d = 0;
        if (a.n < N && a.k < K) {
            const int8_t* from = q + a.e * expert_stride + a.n * stride + a.k;
            int8_t x[8] = {};
            if constexpr (VEC) {
                *reinterpret_cast<uint64_t*>(x) = *reinterpret_cast<const uint64_t*>(from);
            } else {
#pragma unroll
                for (int v = 0; v < 8; ++v)
                    if (a.k + v < K) x[v] = from[v];
            }
#pragma unroll
            for (int v = 0; v < 8; ++v) d |= (uint32_t)(max(-8, min(7, (int)x[v])) & 15) << int4_place(v);
        }
        to[i] = d;
    }
}

// Scales [E, N, groups] -> [E, groups, Np], zeros past N.
template <class T>
__global__ __launch_bounds__(256) void pack_scales_kernel(const T* __restrict__ from, int64_t count, int64_t N,
                                                          int64_t groups, int64_t Np, T* __restrict__ to) {
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < count; i += (int64_t)gridDim.x * 256) {
        const int64_t n = i % Np, row = i / Np, e = row / groups, j = row - e * groups;
        to[i] = n < N ? from[(e * N + n) * groups + j] : (T)0.f;
    }
}

// Scales of a group each by eight lanes: max(amax, 1e-10) / 7. A NaN or an
// infinity makes it one that is not finite.
template <class T>
__global__ __launch_bounds__(256) void int4_scales_kernel(const T* __restrict__ w, int64_t expert_stride,
                                                          int64_t stride, int64_t count, int64_t N, int64_t K,
                                                          int64_t groups, int group, int64_t Np,
                                                          float* __restrict__ to) {
    const int part = threadIdx.x & 7;
    // groups of a channel side by side; the channels past N are zeros
    for (int64_t i = (int64_t)blockIdx.x * 32 + (threadIdx.x >> 3); i < count; i += (int64_t)gridDim.x * 32) {
        const int64_t j = i % groups, c = i / groups, e = c / Np, n = c - e * Np;
        float top = 0.f;
        bool nan = false;
        if (n < N) {
            const T* from = w + e * expert_stride + n * stride;
            const int64_t end = min(K, (j + 1) * group);
            for (int64_t k = j * group + part; k < end; k += 8) {
                const float a = fabsf((float)from[k]);
                nan |= a != a;
                top = fmaxf(top, a);
            }
        }
#pragma unroll
        for (int d = 4; d >= 1; d >>= 1) {
            top = fmaxf(top, __shfl_xor(top, d, 8));
            nan |= __shfl_xor((int)nan, d, 8) != 0;
        }
        if (part == 0)
            to[(e * groups + j) * Np + n] = n >= N ? 0.f : nan ? __builtin_nanf("") : fmaxf(top, 1e-10f) / 7.f;
    }
}

template <class T>
__global__ __launch_bounds__(256) void int4_words_kernel(const T* __restrict__ w, int64_t expert_stride, int64_t stride,
                                                         const float* __restrict__ scale, int64_t words, int64_t N,
                                                         int64_t K, int64_t groups, int shift, int64_t nt, int64_t kt,
                                                         uint32_t* __restrict__ to) {
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < words; i += (int64_t)gridDim.x * 256) {
        const Int4Word a = int4_word(i, nt, kt);
        uint32_t d = 0;
        if (a.n < N && a.k < K) {
            const T* from = w + a.e * expert_stride + a.n * stride;
            const float s = scale[(a.e * groups + (a.k >> shift)) * nt * 16 + a.n];
#pragma unroll
            for (int v = 0; v < 8; ++v)
                if (a.k + v < K) {
                    const float y = rintf((float)from[a.k + v] / s);
                    const int x = y >= -7.f && y <= 7.f ? (int)y : 0;  // others only where s is not finite
                    d |= (uint32_t)(x & 15) << int4_place(v);
                }
        }
        to[i] = d;
    }
}

static unsigned blocks_for(int64_t n, int64_t per) {
    const int64_t b = (n + per - 1) / per;
    return (unsigned)(b < MAX_BLOCKS ? b : MAX_BLOCKS);
}

hipError_t launch_pack_int4(const int8_t* q, int64_t q_expert_stride, int64_t q_stride, const void* scale,
                            int scale_dtype, int64_t E, int64_t N, int64_t K, int group, uint8_t* packed,
                            void* scale_out, hipStream_t s) {
    const int64_t nt = (N + 15) / 16, kt = (K + 127) / 128, words = E * nt * kt * 256;
    const bool vec = ((uint64_t)q | (uint64_t)q_expert_stride | (uint64_t)q_stride | (uint64_t)K) % 8 == 0;
    auto pack = vec ? pack_int4_kernel<true> : pack_int4_kernel<false>;
    hipLaunchKernelGGL(pack, dim3(blocks_for(words, 256)), dim3(256), 0, s, q, q_expert_stride, q_stride, words, N, K, nt,
                       kt, (uint32_t*)packed);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    return by_out_type(scale_dtype, [&](auto t) {
        typedef decltype(t) T;
        const int64_t groups = (K + group - 1) / group, count = E * groups * nt * 16;
        hipLaunchKernelGGL(pack_scales_kernel<T>, dim3(blocks_for(count, 256)), dim3(256), 0, s, (const T*)scale, count,
                           N, groups, nt * 16, (T*)scale_out);
        return hipGetLastError();
    });
}

hipError_t launch_quantize_int4(int dtype, const void* w, int64_t w_expert_stride, int64_t w_stride, int64_t E,
                                int64_t N, int64_t K, int group, uint8_t* packed, float* scale_out, hipStream_t s) {
    const int64_t nt = (N + 15) / 16, kt = (K + 127) / 128, words = E * nt * kt * 256;
    const int64_t groups = (K + group - 1) / group, count = E * groups * nt * 16;
    int shift = 0;
    while (1 << shift < group) ++shift;
    return by_out_type(dtype, [&](auto t) {
        typedef decltype(t) T;
        hipLaunchKernelGGL(int4_scales_kernel<T>, dim3(blocks_for(count, 32)), dim3(256), 0, s, (const T*)w,
                           w_expert_stride, w_stride, count, N, K, groups, group, nt * 16, scale_out);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
        hipLaunchKernelGGL(int4_words_kernel<T>, dim3(blocks_for(words, 256)), dim3(256), 0, s, (const T*)w,
                           w_expert_stride, w_stride, scale_out, words, N, K, groups, shift, nt, kt,
                           (uint32_t*)packed);
        return hipGetLastError();
    });
}

}  // namespace miexp
