// Products of 8-bit integers for any strides, alignment and length
// (mi_experts_int8_matmul).
//
//   out[m, n] = (sum_k a[m, k] b[n, k]) a_scale[m] b_scale[n] + bias[n]
//
// The sum is exact in int32 (K <= 131071), so neither the order of k nor a
// split of it changes a result.
//
// Four waves take a 64 x 64 tile, 64 of K at a time, through registers into
// LDS; 16 bytes that are not aligned, or reach past K, are put together from
// single bytes.
#include "int8_common.hpp"

namespace miexp {

__device__ __forceinline__ v4i bytes16(const int8_t* p, int left, bool aligned) {
    if (aligned && left >= 16) return *reinterpret_cast<const v4i*>(p);
    union { v4i v; int8_t b[16]; } u;
    u.v = (v4i){0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < 16; ++i)
        if (i < left) u.b[i] = p[i];
    return u.v;
}

template <class T>
__global__ __launch_bounds__(256) void int8_general_kernel(Int8Call p, int ntiles, int aligned) {
    constexpr int BM = 64, BN = 64, BK = 64, LD = BK + 16;
    __shared__ __attribute__((aligned(16))) int8_t sa[BM * LD], sb[BN * LD];
    int e, nrows;
    int64_t row0;
    if (!find_tile<BM>(p, blockIdx.x / ntiles, e, row0, nrows)) return;
    const int n0 = (int)(blockIdx.x % ntiles) * BN;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int r = lane & 15, g = lane >> 4;
    const int wm = wave & 1, wn = wave >> 1;

    // loader: thread t copies 16 bytes of tile row t / 4
    const int lr = threadIdx.x >> 2, lc = (threadIdx.x & 3) * 16;
    const int64_t src = lr < nrows ? source_row(p, row0 + lr) : -1;
    const int8_t* pa = src >= 0 ? p.a + src * p.a_stride : nullptr;
    const int8_t* pb = n0 + lr < p.N ? p.b + e * p.b_expert_stride + (n0 + lr) * p.b_stride : nullptr;

    v4i acc[2][2];
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j) acc[i][j] = (v4i){0, 0, 0, 0};
    for (int k0 = 0; k0 < p.K; k0 += BK) {
        const int k = k0 + lc, left = p.K - k;
        const v4i zero = {0, 0, 0, 0};
        const v4i va = pa && left > 0 ? bytes16(pa + k, left, aligned) : zero;
        const v4i vb = pb && left > 0 ? bytes16(pb + k, left, aligned) : zero;
        __syncthreads();
        *reinterpret_cast<v4i*>(sa + lr * LD + lc) = va;
        *reinterpret_cast<v4i*>(sb + lr * LD + lc) = vb;
        __syncthreads();
        v4i fa[2], fb[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            fa[i] = *reinterpret_cast<const v4i*>(sa + (wm * 32 + i * 16 + r) * LD + g * 16);
            fb[i] = *reinterpret_cast<const v4i*>(sb + (wn * 32 + i * 16 + r) * LD + g * 16);
        }
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int j = 0; j < 2; ++j) acc[i][j] = mfma_i8(fb[j], fa[i], acc[i][j]);
    }
    T* out = reinterpret_cast<T*>(p.out);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int m = wm * 32 + i * 16 + r;
        if (m >= nrows) continue;
        const int64_t from = source_row(p, row0 + m);
        const float sam = from >= 0 ? p.a_scale[from] : __builtin_nanf("");
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int v = 0; v < 4; ++v) {
                const int n = n0 + wn * 32 + j * 16 + 4 * g + v;
                if (n >= p.N) continue;
                const float y = (float)acc[i][j][v] * sam * p.b_scale[(int64_t)e * p.N + n];
                out[(row0 + m) * p.out_stride + n] = (T)(y + bias_at(p, n));
            }
    }
}

size_t int8_workspace(int64_t, int64_t, int64_t, int) { return 0; }

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
    const int aligned = (((uint64_t)p.a | (uint64_t)p.b | (uint64_t)p.a_stride | (uint64_t)p.b_stride |
                          (uint64_t)p.b_expert_stride) & 15) == 0;
    const int64_t nt = (a.N + 63) / 64, tiles = max_tiles(a.rows, 64, a.num_experts) * nt;
    const dim3 grid((unsigned)tiles);
    if (a.out_dtype == MI_EXPERTS_F32)
        hipLaunchKernelGGL(int8_general_kernel<float>, grid, dim3(256), 0, s, p, (int)nt, aligned);
    else if (a.out_dtype == MI_EXPERTS_F16)
        hipLaunchKernelGGL(int8_general_kernel<_Float16>, grid, dim3(256), 0, s, p, (int)nt, aligned);
    else
        hipLaunchKernelGGL(int8_general_kernel<__bf16>, grid, dim3(256), 0, s, p, (int)nt, aligned);
    return hipGetLastError();
}

}  // namespace miexp
