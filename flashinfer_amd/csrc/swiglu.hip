// The gate between an expert's two products, with dropout, and its gradient
// (mi_layer_swiglu, mi_layer_swiglu_backward).
//
//   y = v silu(u) m,   silu(u) = u s,  s = 1 / (1 + exp(-u)),  m = keep / (1 - p)
//   dv = g m u s,      du = g m v s (1 + u (1 - s))
//
// x holds v in its first half and u in its second. The mask is not stored: it
// is made again from the seed in the backward pass. One Philox call gives the
// 128 random bits of eight neighbouring columns, 16 bits each, so p is a
// multiple of 1 / 65536 and 1 - p its exact complement. A thread takes eight
// columns of a row.
//
// Memory bounds it: 65536 x 2048 in bf16 with dropout 157 us (5.1 TB/s), its
// gradient 218 (6.1 TB/s); 18006 x 1536 in fp16 36 and 48. Ten rounds of two
// products, sixteen selects and the gate for eight columns stay below that.
// Rows that are not whole vectors of 16 bytes, or not aligned to them, go one
// element at a time: 65536 x 2047 in bf16 415 and 730 us, 18006 x 1535 82 and 145
// (1.8 to 2 TB/s).
#include "layer_common.hpp"

namespace miexp {

constexpr int COLS = 8;  // of a thread: those of one Philox call

// Philox4x32-10 from its definition (Salmon, Moraes, Dror, Shaw: Parallel
// random numbers: as easy as 1, 2, 3; SC 2011): ten rounds of two 32 x 32 bit
// products, whose high words are mixed with the other words and the key, which
// goes on by a constant each round.
__device__ __forceinline__ void philox(uint32_t c0, uint32_t c1, uint64_t seed, uint32_t (&out)[4]) {
    uint32_t x[4] = {c0, c1, 0u, 0u}, k0 = (uint32_t)seed, k1 = (uint32_t)(seed >> 32);
#pragma unroll
    for (int r = 0; r < 10; ++r) {
        const uint64_t a = (uint64_t)x[0] * 0xD2511F53u, b = (uint64_t)x[2] * 0xCD9E8D57u;
        const uint32_t n0 = (uint32_t)(b >> 32) ^ x[1] ^ k0, n2 = (uint32_t)(a >> 32) ^ x[3] ^ k1;
        x[0] = n0;
        x[1] = (uint32_t)b;
        x[2] = n2;
        x[3] = (uint32_t)a;
        k0 += 0x9E3779B9u;
        k1 += 0xBB67AE85u;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) out[i] = x[i];
}

// s = 1 / (1 + exp(-u)). The exponential is 2^(hi + lo) with hi + lo = -u
// log2(e) to twice the precision, the quotient a reciprocal and one Newton
// step. Where 1 + exp(-u) leaves the reciprocal's range the library's
// exponential and a division are taken.
__device__ __forceinline__ void sigmoid(const float (&u)[COLS], float (&s)[COLS]) {
    constexpr float L2E = 1.44269502f, L2E_LO = 1.92596299e-8f, LN2 = 0.693147182f;
    bool far = false;
#pragma unroll
    for (int i = 0; i < COLS; ++i) {
        const float hi = -u[i] * L2E, lo = fmaf(-u[i], L2E_LO, fmaf(-u[i], L2E, -hi));
        float x = __builtin_amdgcn_exp2f(hi);
        x = fmaf(x, lo * LN2, x);
        far |= !(fabsf(u[i]) < 87.f);
        const float d = 1.f + x, rc = __builtin_amdgcn_rcpf(d);
        s[i] = fmaf(fmaf(-rc, d, 1.f), rc, rc);
    }
    if (far) {
#pragma unroll
        for (int i = 0; i < COLS; ++i) s[i] = 1.f / (1.f + expf(-u[i]));
    }
}

struct SwigluCall {
    const void *x, *grad;
    void* out;
    const int32_t* num_rows;
    const uint64_t* seed_ptr;
    uint64_t seed;
    int64_t max_rows, I, x_stride, grad_stride, out_stride;
    uint32_t tile_rows, tile_cols, col_tiles;
    uint32_t threshold;
    float keep_scale;     // 1 / (1 - p)
    int zero_rest;
};

// Eight columns of a row, as vectors or, past the end or off their alignment,
// one at a time.
template <class T, bool VEC>
__device__ __forceinline__ void take(const T* p, int n, float (&v)[COLS]) {
    if constexpr (VEC) {
        constexpr int PER = 16 / (int)sizeof(T);
        typename Vec<T, PER>::type w[COLS / PER];
#pragma unroll
        for (int i = 0; i < COLS / PER; ++i) w[i] = load_once<T, PER>(p + i * PER);
#pragma unroll
        for (int i = 0; i < COLS; ++i) v[i] = (float)w[i / PER][i % PER];
    } else {
#pragma unroll
        for (int i = 0; i < COLS; ++i) v[i] = i < n ? (float)p[i] : 0.f;
    }
}
template <class T, bool VEC>
__device__ __forceinline__ void give(T* p, int n, const float (&v)[COLS]) {
    if constexpr (VEC) {
        constexpr int PER = 16 / (int)sizeof(T);
#pragma unroll
        for (int i = 0; i < COLS / PER; ++i) {
            float w[PER];
#pragma unroll
            for (int e = 0; e < PER; ++e) w[e] = v[i * PER + e];
            store<T, PER>(p + i * PER, w);
        }
    } else {
#pragma unroll
        for (int i = 0; i < COLS; ++i)
            if (i < n) p[i] = (T)v[i];
    }
}

// A workgroup takes `tile_rows` rows of `tile_cols` blocks of eight columns, a
// thread each, and goes on by the grid: units are row tiles x column tiles.
template <class T, bool VEC, bool DROP, bool BACK>
__global__ __launch_bounds__(256) void swiglu_kernel(SwigluCall p) {
    const int64_t rows = p.num_rows ? max((int64_t)0, min(p.max_rows, (int64_t)*p.num_rows)) : p.max_rows;
    const int64_t last = p.zero_rest ? p.max_rows : rows;
    const uint32_t row_in = threadIdx.x / p.tile_cols, block_in = threadIdx.x - row_in * p.tile_cols;
    if (row_in >= p.tile_rows) return;
    uint64_t seed = 0;
    if constexpr (DROP) seed = p.seed_ptr ? *p.seed_ptr : p.seed;
    for (uint32_t unit = blockIdx.x;; unit += gridDim.x) {
        const uint32_t row_tile = unit / p.col_tiles;
        const uint32_t block = (unit - row_tile * p.col_tiles) * p.tile_cols + block_in;
        const int64_t m = (int64_t)row_tile * p.tile_rows + row_in;
        if ((int64_t)row_tile * p.tile_rows >= last) break;
        const int64_t c = (int64_t)block * COLS;
        if (m >= last || c >= p.I) continue;
        const int n = (int)min((int64_t)COLS, p.I - c);
        T* out = (T*)p.out + m * p.out_stride + c;
        if (m >= rows) {
            const float zero[COLS] = {};
            give<T, VEC>(out, n, zero);
            if constexpr (BACK) give<T, VEC>(out + p.I, n, zero);
            continue;
        }
        float v[COLS], u[COLS], g[COLS], s[COLS];
        const T* x = (const T*)p.x + m * p.x_stride + c;
        take<T, VEC>(x, n, v);
        take<T, VEC>(x + p.I, n, u);
        if constexpr (BACK) take<T, VEC>((const T*)p.grad + m * p.grad_stride + c, n, g);
        bool keep[COLS];
        if constexpr (DROP) {
            uint32_t bits[4];
            philox(block, (uint32_t)m, seed, bits);
#pragma unroll
            for (int e = 0; e < COLS; ++e) keep[e] = ((bits[e / 2] >> (16 * (e & 1))) & 0xffffu) >= p.threshold;
        }
        sigmoid(u, s);
        if constexpr (BACK) {
#pragma unroll
            for (int e = 0; e < COLS; ++e) {
                if constexpr (DROP) g[e] *= p.keep_scale;
                const float gs = g[e] * s[e];
                g[e] = gs * u[e];
                u[e] = gs * v[e] * fmaf(u[e], 1.f - s[e], 1.f);
                if constexpr (DROP) {
                    g[e] = keep[e] ? g[e] : 0.f;
                    u[e] = keep[e] ? u[e] : 0.f;
                }
            }
            give<T, VEC>(out, n, g);
            give<T, VEC>(out + p.I, n, u);
        } else {
#pragma unroll
            for (int e = 0; e < COLS; ++e) {
                v[e] *= u[e] * s[e];
                if constexpr (DROP) v[e] = keep[e] ? v[e] * p.keep_scale : 0.f;
            }
            give<T, VEC>(out, n, v);
        }
    }
}

hipError_t launch_swiglu(const mi_layer_swiglu_args& a, bool backward, hipStream_t s) {
    SwigluCall p;
    p.x = a.x;
    p.grad = a.grad;
    p.out = a.out;
    p.num_rows = a.num_rows;
    p.seed_ptr = a.seed_ptr;
    p.seed = a.seed;
    p.max_rows = a.max_rows;
    p.I = a.I;
    p.x_stride = a.x_stride;
    p.grad_stride = a.grad_stride;
    p.out_stride = a.out_stride;
    // Whole rows of up to 256 blocks, as many as 256 threads hold; pieces of longer ones.
    const int64_t blocks = (a.I + COLS - 1) / COLS;
    p.tile_cols = (uint32_t)(blocks < 256 ? blocks : 256);
    p.tile_rows = 256 / p.tile_cols;
    p.col_tiles = (uint32_t)((blocks + 255) / 256);
    const uint32_t threads = (p.tile_rows * p.tile_cols + 63) / 64 * 64;
    const int64_t units = (a.max_rows + p.tile_rows - 1) / p.tile_rows * p.col_tiles;
    p.threshold = (uint32_t)a.threshold;
    p.keep_scale = (float)(65536.0 / (65536 - a.threshold));
    p.zero_rest = a.zero_rest;
    auto go = [&](auto elem) {
        typedef decltype(elem) T;
        constexpr uint64_t PER = 16 / sizeof(T);
        uint64_t bits = (uint64_t)a.x | (uint64_t)a.out, strides = (uint64_t)a.x_stride | (uint64_t)a.out_stride;
        if (backward) bits |= (uint64_t)a.grad, strides |= (uint64_t)a.grad_stride;
        const bool vec = bits % 16 == 0 && strides % PER == 0 && a.I % COLS == 0;
        const dim3 grid((unsigned)(units < MAX_BLOCKS ? units : MAX_BLOCKS));
        auto launch = [&](auto kernel) {
            hipLaunchKernelGGL(kernel, grid, dim3(threads), 0, s, p);
            return hipGetLastError();
        };
        auto pick = [&](auto v, auto d) {
            constexpr bool V = decltype(v)::value != 0, D = decltype(d)::value != 0;
            return backward ? launch(swiglu_kernel<T, V, D, true>) : launch(swiglu_kernel<T, V, D, false>);
        };
        if (a.threshold) return vec ? pick(IntC<1>{}, IntC<1>{}) : pick(IntC<0>{}, IntC<1>{});
        return vec ? pick(IntC<1>{}, IntC<0>{}) : pick(IntC<0>{}, IntC<0>{});
    };
    if (a.dtype == MI_LAYER_F32) return go(float{});
    if (a.dtype == MI_LAYER_F16) return go(_Float16{});
    return go(__bf16{});
}

}  // namespace miexp
