// Rows of floats to int8 with a scale each (mi_experts_quantize_int8), and the
// same after SwiGLU.
//
//   scale[m] = max(amax, 1e-10) / 127,  q = rint(x / scale)
//
// The largest magnitude is found over the bits of |x|, whose order as integers
// is that of the floats with infinities and NaN on top: a row that holds one
// gets a scale that is not finite, and zeros, so that its products are NaN
// instead of numbers made without it.
//
// TX lanes (a wave or a workgroup) take a row. Its first CACHED vectors per
// lane stay in registers between the two passes; longer rows are read (and,
// with SwiGLU, computed) again. Bound by HBM and, with SwiGLU, nearly as much
// by its arithmetic: 8192 x 2048 from bf16 15.2 us (3.3 TB/s), after SwiGLU 22
// (3.8 TB/s); 8192 x 7168 39 to 43 and 64 to 73 us (4.1 to 4.5, 4.0 to 4.6
// TB/s); 130 x 2048 3.4 us. Rows that are no multiples of 16 bytes go by single
// elements: 8192 x 7172 85 and 122 us.
// Zeros for rows that are not in use are written here, too: two fills ahead of
// it made 10.7 us of 5.8 with 64 of 512 rows of 7168 in use.
#include "experts_common.hpp"

namespace miexp {

constexpr float INT8_MAX_F = 127.f;
constexpr float QUANT_FLOOR = 1e-10f;  // scale of an all-zero row: that of quantize_activations

// v = g * u / (1 + exp(-u)). The exponential is 2^(hi + lo) with hi + lo =
// -u log2(e) to twice the precision, the quotient a reciprocal and one Newton
// step: within 6 * 2^-24 of the value, in half the instructions of a library
// exponential and an IEEE division, which bound this kernel. Where 1 + exp(-u)
// leaves the reciprocal's range, or u log2(e) that of fp32, those are what is
// computed.
template <int N>
__device__ __forceinline__ void swiglu(float (&v)[N], const float (&u)[N]) {
    constexpr float L2E = 1.44269502f, L2E_LO = 1.92596299e-8f, LN2 = 0.693147182f;
    float s[N];
    bool far = false;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const float hi = -u[i] * L2E, lo = fmaf(-u[i], L2E_LO, fmaf(-u[i], L2E, -hi));
        float x = __builtin_amdgcn_exp2f(hi);
        x = fmaf(x, lo * LN2, x);
        far |= !(fabsf(u[i]) < 87.f);
        const float d = 1.f + x, rc = __builtin_amdgcn_rcpf(d), q = u[i] * rc;
        s[i] = fmaf(fmaf(-q, d, u[i]), rc, q);
    }
    if (far) {
#pragma unroll
        for (int i = 0; i < N; ++i) s[i] = u[i] / (1.f + expf(-u[i]));
    }
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] *= s[i];
}

template <class T, int N, bool SWIGLU>
__device__ __forceinline__ void quant_input(const T* row, int64_t K, int64_t c, float (&v)[N]) {
    load<T, N>(row + c, v);
    if constexpr (SWIGLU) {
        float u[N];
        load<T, N>(row + K + c, u);
        swiglu(v, u);
    }
}

template <class T, int N, bool SWIGLU, int CACHED, int TX>
__global__ __launch_bounds__(256) void quantize_kernel(const T* __restrict__ x, int64_t x_stride, int64_t M,
                                                       int64_t K, const int32_t* __restrict__ num_rows,
                                                       int zero_rest, int8_t* __restrict__ q, int64_t q_stride,
                                                       float* __restrict__ scale) {
    constexpr int ROWS = 256 / TX;
    __shared__ uint32_t part[4];
    const int lane = threadIdx.x & (TX - 1);
    const int64_t all = M;
    if (num_rows) M = max((int64_t)0, min(M, (int64_t)*num_rows));
    for (int64_t m0 = (int64_t)blockIdx.x * ROWS; m0 < M; m0 += (int64_t)gridDim.x * ROWS) {
        const int64_t m = m0 + threadIdx.x / TX;
        const bool live = m < M;
        const T* row = x + (live ? m : 0) * x_stride;
        float v[CACHED][N];
        uint32_t top = 0;
        auto take = [&](const float (&w)[N]) {
#pragma unroll
            for (int i = 0; i < N; ++i) top = max(top, __float_as_uint(w[i]) & 0x7fffffffu);
        };
        if (live) {
            // all loads before the first use
            typename Vec<T, N>::type g[CACHED], u[CACHED];
#pragma unroll
            for (int i = 0; i < CACHED; ++i) {
                const int64_t c = ((int64_t)i * TX + lane) * N;
                if (c < K) {
                    g[i] = *reinterpret_cast<const typename Vec<T, N>::type*>(row + c);
                    if (SWIGLU) u[i] = *reinterpret_cast<const typename Vec<T, N>::type*>(row + K + c);
                }
            }
#pragma unroll
            for (int i = 0; i < CACHED; ++i) {
                if (((int64_t)i * TX + lane) * N >= K) continue;
#pragma unroll
                for (int e = 0; e < N; ++e) v[i][e] = element<T, N>(g[i], e);
                if constexpr (SWIGLU) {
                    float w[N];
#pragma unroll
                    for (int e = 0; e < N; ++e) w[e] = element<T, N>(u[i], e);
                    swiglu(v[i], w);
                }
                take(v[i]);
            }
            for (int64_t c = ((int64_t)CACHED * TX + lane) * N; c < K; c += (int64_t)TX * N) {
                float w[N];
                quant_input<T, N, SWIGLU>(row, K, c, w);
                take(w);
            }
        }
#pragma unroll
        for (int d = 32; d >= 1; d >>= 1) top = max(top, (uint32_t)__shfl_xor((int)top, d));
        if constexpr (TX > 64) {
            if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = top;
            __syncthreads();
            top = max(max(part[0], part[1]), max(part[2], part[3]));
            __syncthreads();
        }
        if (!live) continue;
        const bool finite = top < 0x7f800000u;
        const float amax = __uint_as_float(top);
        const float s = finite ? fmaxf(amax, QUANT_FLOOR) / INT8_MAX_F : amax;
        const float inverse = 1.f / s;  // finite: s >= 7.8e-13
        auto put = [&](int64_t c, const float (&w)[N]) {
            int8_t b[N];
            if constexpr (SWIGLU) {
                // rint(w / s) by a product with 1 / s, whose error is below
                // 127 * 2^-22 = 3.1e-5, unless that could change a rounding.
                // (The plain quantiser has the time for its divisions: 41
                // against 49 us at 8192 x 7168; here it is 80 against 63.)
                float x[N];
                bool tie = false;
#pragma unroll
                for (int i = 0; i < N; ++i) {
                    const float y = w[i] * inverse;
                    x[i] = rintf(y);
                    tie |= !(fabsf(y - x[i]) < 0.4999f);
                }
                if (tie) {
#pragma unroll
                    for (int i = 0; i < N; ++i) x[i] = finite ? rintf(w[i] / s) : 0.f;
                }
#pragma unroll
                for (int i = 0; i < N; ++i) b[i] = (int8_t)(int)x[i];
            } else {
#pragma unroll
                for (int i = 0; i < N; ++i) b[i] = finite ? (int8_t)(int)rintf(w[i] / s) : (int8_t)0;
            }
            if constexpr (N == 8)
                *reinterpret_cast<uint2*>(q + m * q_stride + c) = *reinterpret_cast<const uint2*>(b);
            else if constexpr (N == 4)
                *reinterpret_cast<uint32_t*>(q + m * q_stride + c) = *reinterpret_cast<const uint32_t*>(b);
            else
                q[m * q_stride + c] = b[0];
        };
#pragma unroll
        for (int i = 0; i < CACHED; ++i) {
            const int64_t c = ((int64_t)i * TX + lane) * N;
            if (c < K) put(c, v[i]);
        }
        for (int64_t c = ((int64_t)CACHED * TX + lane) * N; c < K; c += (int64_t)TX * N) {
            float w[N];
            quant_input<T, N, SWIGLU>(row, K, c, w);
            put(c, w);
        }
        if (lane == 0) scale[m] = s;
    }
    if (!zero_rest) return;
    for (int64_t m = M + (int64_t)blockIdx.x * ROWS + threadIdx.x / TX; m < all; m += (int64_t)gridDim.x * ROWS) {
        for (int64_t c = (int64_t)lane * N; c < K; c += (int64_t)TX * N) {
            if constexpr (N == 8)
                *reinterpret_cast<uint2*>(q + m * q_stride + c) = make_uint2(0, 0);
            else if constexpr (N == 4)
                *reinterpret_cast<uint32_t*>(q + m * q_stride + c) = 0;
            else
                q[m * q_stride + c] = 0;
        }
        if (lane == 0) scale[m] = 0.f;
    }
}

struct Yes { static constexpr bool value = true; };
struct No { static constexpr bool value = false; };

hipError_t launch_quantize(int dtype, const void* x, int64_t x_stride, int64_t M, int64_t K, bool swiglu,
                           const int32_t* num_rows, bool zero_rest, int8_t* q, int64_t q_stride,
                           float* scale, hipStream_t s) {
    auto go = [&](auto elem, auto wide) {
        typedef decltype(elem) E;
        constexpr int N = decltype(wide)::value ? 16 / (int)sizeof(E) : 1;
        auto launch = [&](auto kernel, int rows) {
            const int64_t b = (M + rows - 1) / rows;
            hipLaunchKernelGGL(kernel, dim3((unsigned)(b < MAX_BLOCKS ? b : MAX_BLOCKS)), dim3(256), 0, s,
                               (const E*)x, x_stride, M, K, num_rows, (int)zero_rest, q, q_stride, scale);
            return hipGetLastError();
        };
        // A wave for a short row, and where there are rows enough to fill the
        // chip with waves; a workgroup for a row else (8192 x 2048: 14.7 against
        // 16.9 us; 4096 x 4096: 16.7 against 14.2).
        if (K <= 128 * N && (K <= 64 * N || M >= 512))
            return swiglu ? launch(quantize_kernel<E, N, true, 2, 64>, 4) : launch(quantize_kernel<E, N, false, 2, 64>, 4);
        if (K <= 256 * N && M >= 2048)
            return swiglu ? launch(quantize_kernel<E, N, true, 4, 64>, 4) : launch(quantize_kernel<E, N, false, 4, 64>, 4);
        return swiglu ? launch(quantize_kernel<E, N, true, 4, 256>, 1) : launch(quantize_kernel<E, N, false, 4, 256>, 1);
    };
    const uint64_t size = dtype == MI_EXPERTS_F32 ? 4 : 2;
    const bool wide = (((uint64_t)x_stride | (uint64_t)K) * size) % 16 == 0 && (uint64_t)x % 16 == 0 &&
                      ((uint64_t)q | (uint64_t)q_stride) % 8 == 0;
    if (dtype == MI_EXPERTS_F32) return wide ? go(float{}, Yes{}) : go(float{}, No{});
    if (dtype == MI_EXPERTS_F16) return wide ? go(_Float16{}, Yes{}) : go(_Float16{}, No{});
    return wide ? go(__bf16{}, Yes{}) : go(__bf16{}, No{});
}

}  // namespace miexp
