// Token rows to expert order and back (mi_experts_permute, _unpermute,
// _unpermute_backward).
//
// All three go by token: a token's row and its k places are read once, and the
// k rows that belong to it are written (or gathered) from there, so the
// smaller side of the traffic crosses HBM once and no row index has to be
// inverted. The sums over a token's slots and over a row's columns run in
// fp32 in a fixed order; no atomics.
//
// All are bound by HBM. On MI355X, where a large copy reaches 4.7 TB/s, 8192
// tokens x 8 rows of 7168 bf16: permute 218 us (4.9 TB/s), unpermute 195 us
// (5.4), its gradients 400 us (5.0); one token: 2.8 us. Rows are read past the
// caches (unpermute 235 us without).
//
// tx = 2^tx_log lanes share a token (as many as its row has vectors, at most
// a workgroup), so short rows still fill the waves. From 64 lanes on a wave has
// one token (ONE): its places, weights and whether a slot is local are then
// scalar, and slots of other shards cost a scalar branch.
#include "experts_common.hpp"

namespace miexp {

constexpr int THREADS = 256;
constexpr int KG = 8;  // slots of a token handled together

inline int lanes_log(int64_t vectors) {
    int l = 0;
    while (l < 8 && (1ll << l) < vectors) ++l;
    return l;
}

// The token of this thread in a group of THREADS >> tx_log.
template <bool ONE>
__device__ __forceinline__ int token_in_group(int tx_log) {
    const int t = threadIdx.x >> tx_log;
    return ONE ? __builtin_amdgcn_readfirstlane(t) : t;
}

// Workgroups over T tokens and `chunks` column chunks, fewer than 2^32 threads.
inline dim3 grid_for(int64_t T, int tx_log, int64_t chunks) {
    const int64_t b = (T + (THREADS >> tx_log) - 1) / (THREADS >> tx_log), most = ((int64_t)1 << 23) / chunks;
    return dim3((unsigned)(b < most ? b : most), (unsigned)chunks);
}

// Rows that all together exceed the 256 MB of the last cache are stored past
// it: they would be gone before their reader comes, and what they push out has
// to be written back meanwhile (permute and its gradient, 3001 x 6 rows of
// 4096 fp32: 53 + 100 us cached, 57 + 62 past it; 8192 x 8 of 7168 bf16 184 +
// 258 against 219 + 192). Smaller ones are stored faster into it (8000 rows of 7168
// bf16 18.5 us, 23.5 past it; the gradients of 3001 x 6 of 4096 fp16 53 and 57)
// and stay for their reader.
inline bool streams(int64_t bytes) { return bytes > (int64_t)256 << 20; }

// Rows of slots j0 .. j0 + KG - 1 of token t (-1 past the k of it), all loaded
// before the first is used: loads and stores of rows in between would be
// waited for with them, memory operations completing in order.
__device__ __forceinline__ void rows_of(const int32_t* row_of_slot, int64_t t, int k, int j0, int (&row)[KG]) {
#pragma unroll
    for (int j = 0; j < KG; ++j) row[j] = row_of_slot[t * k + min(j0 + j, k - 1)];
#pragma unroll
    for (int j = 0; j < KG; ++j)
        if (j0 + j >= k) row[j] = -1;
}

// V: the unit that moves, as wide as row length, strides and addresses allow.
template <class V, bool ONE, bool STREAM>
__global__ __launch_bounds__(THREADS) void permute_kernel(const char* __restrict__ x, int64_t x_stride,
                                                          int64_t T, int k, int64_t vectors,
                                                          const int32_t* __restrict__ row_of_slot,
                                                          const int32_t* __restrict__ num_rows,
                                                          char* __restrict__ rows, int64_t rows_stride,
                                                          int zero_rest, int tx_log) {
    const int tx = 1 << tx_log;
    const int64_t R = T * k;
    const int64_t local = min((int64_t)*num_rows, R);
    const int64_t v = (int64_t)blockIdx.y * tx + (threadIdx.x & (tx - 1));
    if (v >= vectors) return;
    for (int64_t t = (int64_t)blockIdx.x * (THREADS >> tx_log) + token_in_group<ONE>(tx_log); t < T;
         t += (int64_t)gridDim.x * (THREADS >> tx_log)) {
        const V val = reinterpret_cast<const V*>(x + t * x_stride)[v];
        for (int j0 = 0; j0 < k; j0 += KG) {
            int row[KG];
            rows_of(row_of_slot, t, k, j0, row);
#pragma unroll
            for (int j = 0; j < KG; ++j) {
                if (row[j] >= 0 && row[j] < local)
                    put<STREAM>(&reinterpret_cast<V*>(rows + row[j] * rows_stride)[v], val);
                else if (zero_rest && row[j] >= 0 && row[j] < R)
                    put<STREAM>(&reinterpret_cast<V*>(rows + row[j] * rows_stride)[v], V{});
            }
        }
    }
}

hipError_t launch_permute(const void* x, int64_t x_stride, int64_t T, int k, int64_t row_bytes,
                          const int32_t* row_of_slot, const int32_t* num_rows, void* rows,
                          int64_t rows_stride, bool zero_rest, hipStream_t s) {
    const uint64_t bits = (uint64_t)x | (uint64_t)rows | (uint64_t)x_stride | (uint64_t)rows_stride |
                          (uint64_t)row_bytes;
    auto go = [&](auto unit) {
        typedef decltype(unit) V;
        const int64_t vectors = row_bytes / (int64_t)sizeof(V);
        const int tx_log = lanes_log(vectors);
        const dim3 grid = grid_for(T, tx_log, (vectors + (1 << tx_log) - 1) >> tx_log);
        const bool stream = streams(T * k * row_bytes);
        const auto kernel = tx_log >= 6 ? (stream ? permute_kernel<V, true, true> : permute_kernel<V, true, false>)
                                        : (stream ? permute_kernel<V, false, true> : permute_kernel<V, false, false>);
        hipLaunchKernelGGL(kernel, grid, dim3(THREADS), 0, s, (const char*)x, x_stride, T, k, vectors, row_of_slot,
                           num_rows, (char*)rows, rows_stride, (int)zero_rest, tx_log);
        return hipGetLastError();
    };
    if (bits % 16 == 0) return go(v4i{});
    if (bits % 8 == 0) return go((uint64_t)0);
    if (bits % 4 == 0) return go((uint32_t)0);
    if (bits % 2 == 0) return go((uint16_t)0);
    return go((uint8_t)0);
}

template <class T, int N, bool WEIGHTED, bool ONE>
__global__ __launch_bounds__(THREADS) void unpermute_kernel(const T* __restrict__ rows, int64_t rows_stride,
                                                            int64_t tokens, int k, int64_t H,
                                                            const int32_t* __restrict__ row_of_slot,
                                                            const int32_t* __restrict__ num_rows,
                                                            const float* __restrict__ weights,
                                                            T* __restrict__ out, int64_t out_stride,
                                                            int tx_log) {
    const int tx = 1 << tx_log;
    const int64_t local = min((int64_t)*num_rows, tokens * k);
    const int64_t c = ((int64_t)blockIdx.y * tx + (threadIdx.x & (tx - 1))) * N;
    if (c >= H) return;
    for (int64_t t = (int64_t)blockIdx.x * (THREADS >> tx_log) + token_in_group<ONE>(tx_log); t < tokens;
         t += (int64_t)gridDim.x * (THREADS >> tx_log)) {
        float acc[N];
#pragma unroll
        for (int i = 0; i < N; ++i) acc[i] = 0.f;
        for (int j0 = 0; j0 < k; j0 += KG) {
            int row[KG];
            float w[KG];
            rows_of(row_of_slot, t, k, j0, row);
            if (WEIGHTED) {
#pragma unroll
                for (int j = 0; j < KG; ++j) w[j] = weights[t * k + min(j0 + j, k - 1)];
            }
            typename Vec<T, N>::type v[KG];
            bool on[KG];
#pragma unroll
            for (int j = 0; j < KG; ++j) {
                on[j] = row[j] >= 0 && row[j] < local;
                if (on[j]) v[j] = load_once<T, N>(rows + row[j] * rows_stride + c);
            }
#pragma unroll
            for (int j = 0; j < KG; ++j)
                if (on[j]) {
#pragma unroll
                    for (int i = 0; i < N; ++i) {
                        const float x = element<T, N>(v[j], i);
                        acc[i] = WEIGHTED ? fmaf(w[j], x, acc[i]) : acc[i] + x;
                    }
                }
        }
        store<T, N>(out + t * out_stride + c, acc);
    }
}

// Gradients of a token's rows and weights: its tx lanes walk the columns, each
// lane keeps one partial product sum per slot, and the sums meet at the end.
template <class T, int N, bool ONE, bool STREAM>
__global__ __launch_bounds__(THREADS) void unpermute_backward_kernel(
    const T* __restrict__ grad, int64_t grad_stride, const T* __restrict__ rows, int64_t rows_stride,
    int64_t tokens, int k, int64_t H, const int32_t* __restrict__ row_of_slot,
    const int32_t* __restrict__ num_rows, const float* __restrict__ weights, T* __restrict__ grad_rows,
    int64_t grad_rows_stride, int zero_rest, float* __restrict__ grad_weights, int tx_log) {
    __shared__ float part[THREADS / 64][KG];
    const int tx = 1 << tx_log, lane = threadIdx.x & (tx - 1);
    const int64_t R = tokens * k;
    const int64_t local = min((int64_t)*num_rows, R);
    const int64_t per = THREADS >> tx_log;
    // the same number of rounds for all threads: they meet at the barriers
    for (int64_t t0 = (int64_t)blockIdx.x * per; t0 < tokens; t0 += (int64_t)gridDim.x * per) {
        const int64_t t = t0 + token_in_group<ONE>(tx_log);
        const bool live = t < tokens;
        for (int j0 = 0; j0 < k; j0 += KG) {
            int row[KG];
            float w[KG], dot[KG];
            rows_of(row_of_slot, min(t, tokens - 1), k, j0, row);
#pragma unroll
            for (int j = 0; j < KG; ++j) {
                if (!live || row[j] >= R) row[j] = -1;
                w[j] = weights ? weights[min(t, tokens - 1) * k + min(j0 + j, k - 1)] : 1.f;
                dot[j] = 0.f;
            }
            if (live) {
                for (int64_t c = (int64_t)lane * N; c < H; c += (int64_t)tx * N) {
                    float g[N];
                    load<T, N>(grad + t * grad_stride + c, g);
                    typename Vec<T, N>::type v[KG];
                    if (grad_weights) {
#pragma unroll
                        for (int j = 0; j < KG; ++j)
                            if (row[j] >= 0 && row[j] < local) v[j] = load_once<T, N>(rows + row[j] * rows_stride + c);
                    }
#pragma unroll
                    for (int j = 0; j < KG; ++j) {
                        const bool on = row[j] >= 0 && row[j] < local;
                        if (row[j] < 0 || !(on || zero_rest)) continue;
                        if (on && grad_weights) {
#pragma unroll
                            for (int i = 0; i < N; ++i) dot[j] = fmaf(g[i], element<T, N>(v[j], i), dot[j]);
                        }
                        if (grad_rows) {
                            float d[N];
#pragma unroll
                            for (int i = 0; i < N; ++i) d[i] = on ? w[j] * g[i] : 0.f;
                            store<T, N, STREAM>(grad_rows + row[j] * grad_rows_stride + c, d);
                        }
                    }
                }
            }
            if (!grad_weights) continue;
            for (int d = min(tx, 64) >> 1; d >= 1; d >>= 1)
#pragma unroll
                for (int j = 0; j < KG; ++j) dot[j] += __shfl_xor(dot[j], d);
            if (tx > 64) {
                if ((threadIdx.x & 63) == 0)
#pragma unroll
                    for (int j = 0; j < KG; ++j) part[threadIdx.x >> 6][j] = dot[j];
                __syncthreads();
                const int w0 = (threadIdx.x >> tx_log) * (tx >> 6);
#pragma unroll
                for (int j = 0; j < KG; ++j) {
                    dot[j] = 0.f;
                    for (int w1 = 0; w1 < tx >> 6; ++w1) dot[j] += part[w0 + w1][j];
                }
                __syncthreads();
            }
            if (live && lane == 0)
#pragma unroll
                for (int j = 0; j < KG; ++j)
                    if (j0 + j < k) grad_weights[t * k + j0 + j] = dot[j];
        }
    }
}

// Calls go(T{}, IntC<N>{}) with vectors of 16 bytes, or single elements where the
// row length, strides (in elements) or addresses are no multiples of 16 bytes:
// 8192 x 8 rows of 7168 bf16 196 us, its gradients 398, of 7172 680 and 1058.
// (permute, whose units go by halves: 183, 7172 319, 7170 392, 7169 542.)
template <class F>
hipError_t by_type(int dtype, uint64_t elems, uint64_t addresses, F go) {
    const int size = dtype == MI_EXPERTS_F32 ? 4 : 2;
    const bool wide = (elems * size) % 16 == 0 && addresses % 16 == 0;
    if (dtype == MI_EXPERTS_F32) return wide ? go(float{}, IntC<4>{}) : go(float{}, IntC<1>{});
    if (dtype == MI_EXPERTS_F16) return wide ? go(_Float16{}, IntC<8>{}) : go(_Float16{}, IntC<1>{});
    return wide ? go(__bf16{}, IntC<8>{}) : go(__bf16{}, IntC<1>{});
}

hipError_t launch_unpermute(int dtype, const void* rows, int64_t rows_stride, int64_t T, int k, int64_t H,
                            const int32_t* row_of_slot, const int32_t* num_rows, const float* weights,
                            void* out, int64_t out_stride, hipStream_t s) {
    return by_type(dtype, (uint64_t)rows_stride | (uint64_t)out_stride | (uint64_t)H,
                   (uint64_t)rows | (uint64_t)out, [&](auto elem, auto width) {
        typedef decltype(elem) E;
        constexpr int N = decltype(width)::value;
        const int64_t vectors = (H + N - 1) / N;
        const int tx_log = lanes_log(vectors);
        const dim3 grid = grid_for(T, tx_log, (vectors + (1 << tx_log) - 1) >> tx_log);
        const auto kernel = weights ? (tx_log >= 6 ? unpermute_kernel<E, N, true, true> : unpermute_kernel<E, N, true, false>)
                                    : (tx_log >= 6 ? unpermute_kernel<E, N, false, true> : unpermute_kernel<E, N, false, false>);
        hipLaunchKernelGGL(kernel, grid, dim3(THREADS), 0, s, (const E*)rows, rows_stride, T, k, H, row_of_slot,
                           num_rows, weights, (E*)out, out_stride, tx_log);
        return hipGetLastError();
    });
}

hipError_t launch_unpermute_backward(int dtype, const void* grad, int64_t grad_stride, const void* rows,
                                     int64_t rows_stride, int64_t T, int k, int64_t H,
                                     const int32_t* row_of_slot, const int32_t* num_rows,
                                     const float* weights, void* grad_rows, int64_t grad_rows_stride,
                                     bool zero_rest, float* grad_weights, hipStream_t s) {
    const uint64_t elems = (uint64_t)grad_stride | (uint64_t)H | (grad_weights ? (uint64_t)rows_stride : 0) |
                           (grad_rows ? (uint64_t)grad_rows_stride : 0);
    const uint64_t addr = (uint64_t)grad | (grad_weights ? (uint64_t)rows : 0) | (uint64_t)grad_rows;
    return by_type(dtype, elems, addr, [&](auto elem, auto width) {
        typedef decltype(elem) E;
        constexpr int N = decltype(width)::value;
        const int tx_log = lanes_log((H + N - 1) / N);
        const bool stream = streams(T * k * H * (int64_t)sizeof(E));
        const auto kernel =
            tx_log >= 6
                ? (stream ? unpermute_backward_kernel<E, N, true, true> : unpermute_backward_kernel<E, N, true, false>)
                : (stream ? unpermute_backward_kernel<E, N, false, true> : unpermute_backward_kernel<E, N, false, false>);
        hipLaunchKernelGGL(kernel, grid_for(T, tx_log, 1), dim3(THREADS), 0, s, (const E*)grad, grad_stride,
                           (const E*)rows, rows_stride, T, k, H, row_of_slot, num_rows, weights, (E*)grad_rows,
                           grad_rows_stride, (int)zero_rest, grad_weights, tx_log);
        return hipGetLastError();
    });
}

}  // namespace miexp
