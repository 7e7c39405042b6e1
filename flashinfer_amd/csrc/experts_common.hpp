// Shared by the expert operators (libmi_experts.so): element types, vector
// loads, and the tables that place slots at rows.
#pragma once

#include <hip/hip_runtime.h>
#include <stddef.h>
#include <stdint.h>

#include "../../include/mi_experts.h"

namespace miexp {

typedef int v4i __attribute__((ext_vector_type(4)));

// Workgroups of the row-moving kernels are capped and loop: a launch holds
// fewer than 2^32 threads.
constexpr int64_t MAX_BLOCKS = 1 << 20;

template <int DT> struct Elem;
template <> struct Elem<MI_EXPERTS_BF16> { typedef __bf16 type; };
template <> struct Elem<MI_EXPERTS_F16> { typedef _Float16 type; };
template <> struct Elem<MI_EXPERTS_F32> { typedef float type; };

// N consecutive elements at p as one load or store (p aligned to their size).
template <class T, int N> struct Vec { typedef T type __attribute__((ext_vector_type(N))); };
template <class T> struct Vec<T, 1> { typedef T type; };

template <class T, int N>
__device__ __forceinline__ float element(const typename Vec<T, N>::type& v, int i) {
    if constexpr (N == 1) return (float)v;
    else return (float)v[i];
}

// N elements that are read once: the load leaves nothing in the caches.
template <class T, int N>
__device__ __forceinline__ typename Vec<T, N>::type load_once(const T* p) {
    return __builtin_nontemporal_load(reinterpret_cast<const typename Vec<T, N>::type*>(p));
}

template <class T, int N>
__device__ __forceinline__ void load(const T* p, float (&v)[N]) {
    if constexpr (N == 1) {
        v[0] = (float)*p;
    } else {
        const auto w = *reinterpret_cast<const typename Vec<T, N>::type*>(p);
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = (float)w[i];
    }
}

// STREAM: the store passes the caches by. (A run-time choice would not do: the
// compiler makes one plain store of two that differ in this alone.)
template <bool STREAM, class V>
__device__ __forceinline__ void put(V* p, V v) {
    if constexpr (STREAM)
        __builtin_nontemporal_store(v, p);
    else
        *p = v;
}

template <class T, int N, bool STREAM = false>
__device__ __forceinline__ void store(T* p, const float (&v)[N]) {
    typename Vec<T, N>::type w;
    if constexpr (N == 1) {
        w = (T)v[0];
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) w[i] = (T)v[i];
    }
    put<STREAM>(reinterpret_cast<typename Vec<T, N>::type*>(p), w);
}

template <int N> struct IntC { static constexpr int value = N; };

// Launchers (host).
hipError_t launch_sort(const int32_t* ids, int64_t T, int k, int E, int64_t offset, int32_t* offsets,
                       int32_t* token_of_row, int32_t* row_of_slot, int32_t* counts, hipStream_t s);
int64_t sort_chunks(int64_t slots);  // 0: one workgroup sorts alone, no workspace
hipError_t launch_permute(const void* x, int64_t x_stride, int64_t T, int k, int64_t row_bytes,
                          const int32_t* row_of_slot, const int32_t* num_rows, void* rows,
                          int64_t rows_stride, bool zero_rest, hipStream_t s);
hipError_t launch_unpermute(int dtype, const void* rows, int64_t rows_stride, int64_t T, int k, int64_t H,
                            const int32_t* row_of_slot, const int32_t* num_rows, const float* weights,
                            void* out, int64_t out_stride, hipStream_t s);
hipError_t launch_unpermute_backward(int dtype, const void* grad, int64_t grad_stride, const void* rows,
                                     int64_t rows_stride, int64_t T, int k, int64_t H,
                                     const int32_t* row_of_slot, const int32_t* num_rows,
                                     const float* weights, void* grad_rows, int64_t grad_rows_stride,
                                     bool zero_rest, float* grad_weights, hipStream_t s);
hipError_t launch_quantize(int dtype, const void* x, int64_t x_stride, int64_t M, int64_t K, bool swiglu,
                           const int32_t* num_rows, bool zero_rest, int8_t* q, int64_t q_stride, float* scale,
                           hipStream_t s);
hipError_t launch_int8_matmul(const mi_experts_int8_args& a, hipStream_t s);
size_t int8_workspace(int64_t rows, int64_t N, int64_t K, int E);

}  // namespace miexp
