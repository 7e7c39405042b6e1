// Products of a few rows with 4-bit weights: what bounds them is reading the
// weights once.
//
// A workgroup takes 16 rows (of one expert) and NT tiles of 16 channels, its
// eight waves every eighth tile of 128 values of K each. A lane loads its 16
// bytes of a weight tile, its scales and its pieces of the rows from memory
// into registers: nothing goes through LDS, no wave waits for another before
// the end, and the loads of two batches of tiles are on their way before the first is
// used. The waves' sums meet in LDS. Any number of rows is right here, as all
// others' offsets are 64 bits: this kernel also takes what does not fit those
// of int4_tile.hip.
#include "int4_common.hpp"

namespace miexp {

constexpr int ROW_KS = 8;

template <class XT, class ST, int GS, int NT>
__global__ __launch_bounds__(64 * ROW_KS, 2) void int4_row_kernel(Int4Call p, int ntiles, int vec) {
    typedef Operand<XT> Op;
    typedef typename Op::frag frag;
    constexpr int G = 4 / GS;           // scales of a tile
    constexpr int U = G == 4 ? 2 : 3;  // tiles in a batch: two batches fill the registers
    typedef ST s4 __attribute__((ext_vector_type(4)));
    __shared__ v4f sums[ROW_KS][NT][64];
    const int lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4;
    const int ks = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int64_t total = (int64_t)count_tiles<16>(p) * ntiles;
    for (int64_t tile = blockIdx.x; tile < total; tile += gridDim.x) {
        int e, nrows;
        int64_t row0;
        const int mt = (int)(tile / ntiles), n_first = (int)(tile - (int64_t)mt * ntiles) * NT;
        find_tile<16>(p, mt, e, row0, nrows);
        const int64_t from = max(source_row(p, row0 + min(r, nrows - 1)), (int64_t)0);
        const XT* x = (const XT*)p.x + from * p.x_stride;
        const ST* scale = (const ST*)p.scale + e * p.scale_expert + 4 * g;
        const int last_n = (p.N + 15) / 16 - 1;
        const uint8_t* w[NT];
#pragma unroll
        for (int n = 0; n < NT; ++n)
            w[n] = p.w + e * p.w_expert + (int64_t)min(n_first + n, last_n) * p.KT * 1024 + lane * 16;
        v4f acc[NT];
#pragma unroll
        for (int n = 0; n < NT; ++n) acc[n] = (v4f){0.f, 0.f, 0.f, 0.f};
        struct Batch {
            v4u w[U][NT];
            v4u x[U][4];
            s4 s[U][NT][G];
        };
        auto fetch = [&](Batch& b, int k0) __attribute__((always_inline)) {
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int kt = min(k0 + u * ROW_KS, p.KT - 1);
#pragma unroll
                for (int n = 0; n < NT; ++n)
                    b.w[u][n] = __builtin_nontemporal_load(reinterpret_cast<const v4u*>(w[n] + (int64_t)kt * 1024));
#pragma unroll
                for (int i = 0; i < 4; ++i)  // past K: any value, cut below
                    b.x[u][i] = *reinterpret_cast<const v4u*>(x + min(kt * 128 + 32 * i + 8 * g, p.K - 8));
#pragma unroll
                for (int j = 0; j < G; ++j) {
                    const int row = min(kt * 128 + j * (32 * GS), p.K - 1) >> p.group_shift;
#pragma unroll
                    for (int n = 0; n < NT; ++n)
                        b.s[u][n][j] = *reinterpret_cast<const s4*>(scale + (int64_t)row * p.Np +
                                                                    min(n_first + n, last_n) * 16);
                }
            }
        };
        auto use = [&](Batch& b, int k0) __attribute__((always_inline)) {
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int kt = k0 + u * ROW_KS;
                if (kt >= p.KT) break;
                if (kt * 128 + 128 > p.K) {
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        if (kt * 128 + 32 * i + 8 * g >= p.K) b.x[u][i] = (v4u){0, 0, 0, 0};
                }
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int j = 0; j < G; ++j) {
                        v4f t = (v4f){0.f, 0.f, 0.f, 0.f};
#pragma unroll
                        for (int i = j * GS; i < j * GS + GS; ++i)
                            t = Op::mfma(Op::weights(b.w[u][n][i]), __builtin_bit_cast(frag, b.x[u][i]), t);
#pragma unroll
                        for (int v = 0; v < 4; ++v)
                            acc[n][v] = fmaf((float)b.s[u][n][j][v] * Op::UNIT, t[v], acc[n][v]);
                    }
            }
        };
        Batch a, b;
        fetch(a, ks);
        for (int k0 = ks; k0 < p.KT; k0 += 2 * U * ROW_KS) {
            if (k0 + U * ROW_KS < p.KT) fetch(b, k0 + U * ROW_KS);
            use(a, k0);
            if (k0 + U * ROW_KS >= p.KT) break;
            if (k0 + 2 * U * ROW_KS < p.KT) fetch(a, k0 + 2 * U * ROW_KS);
            use(b, k0 + U * ROW_KS);
        }
#pragma unroll
        for (int n = 0; n < NT; ++n) sums[ks][n][lane] = acc[n];
        __syncthreads();
        if (threadIdx.x < 64 * NT) {
            const int n = threadIdx.x >> 6;
            v4f y = sums[0][n][lane];
#pragma unroll
            for (int i = 1; i < ROW_KS; ++i) y += sums[i][n][lane];
            if (r < nrows) store_sums(p, row0 + r, (n_first + n) * 16 + 4 * g, vec, y);
        }
        __syncthreads();
    }
    zero_rest_any(p, vec);
}

hipError_t launch_int4_row(const Int4Call& p, int x_dtype, int scale_dtype, bool vec, hipStream_t s) {
    return by_int4_types(x_dtype, scale_dtype, 1 << p.group_shift, [&](auto x, auto sc, auto gs) {
        const int ntiles = (p.N + 15) / 16;
        const int64_t tiles = max_tiles(p.rows, 16, p.E) * ntiles;
        hipLaunchKernelGGL((int4_row_kernel<decltype(x), decltype(sc), decltype(gs)::value, 1>),
                           dim3((unsigned)(tiles < 4096 ? tiles : 4096)), dim3(64 * ROW_KS), 0, s, p, ntiles, (int)vec);
        return hipGetLastError();
    });
}

}  // namespace miexp
