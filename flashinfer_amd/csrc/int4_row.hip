// Products of a few rows with 4-bit weights: what bounds them is reading the
// weights once, and with few workgroups the length of a workgroup's chain of
// loads.
//
// A workgroup takes 4 XC rows (of one expert) and 16 channels, its eight waves
// every eighth tile of 128 values of K each. A wave copies its weight tiles, the
// rows' values that go with them and the scales into LDS slots of its own, D
// tiles ahead of their use, and waits for nothing but its own copies; the waves'
// sums meet at the end. Addresses are 64 bits for each lane, so this kernel also
// takes what the 32-bit offsets of int4_tile.hip do not reach, with 16 rows.
//
// 1 x 4096 x 7168 7.1 to 7.7 us, 6.1 on the GPU: 2.7 of a launch that does nothing,
// 1.6 of making weights and what the loads of 14.7 MB take beside it. (Loads into
// registers instead: 8.9, and 13.2 with 16 rows, here 8.8.)
#include "int4_common.hpp"
#include "lds_copy.hpp"

namespace miexp {

using mimoe::g2l16;
using mimoe::g2l4;

constexpr int ROW_KS = 8;

// Waits until at most LD * r copies are in flight, for r up to R.
template <int LD, int R>
__device__ __forceinline__ void wait_steps(int r) {
    if constexpr (R == 0) {
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    } else {
        if (r >= R)
            asm volatile("s_waitcnt vmcnt(%0)" ::"n"(LD * R) : "memory");
        else
            wait_steps<LD, R - 1>(r);
    }
}

template <class XT, class ST, int GS, int XC, int D>
__global__ __launch_bounds__(64 * ROW_KS) void int4_row_kernel(Int4Call p, int ntiles, int vec) {
    typedef Operand<XT> Op;
    typedef typename Op::frag frag;
    typedef ST s4 __attribute__((ext_vector_type(4)));
    constexpr int G = 4 / GS, BM = 4 * XC, LD = 1 + XC + 1;
    constexpr int X = 1024, S = X + XC * 1024, SLOT = S + 256;  // weights, rows, scales: G * 16, at most 256 bytes
    static_assert(G * 16 * sizeof(ST) <= 256 && LD * (D - 1) < 64, "slots");
    __shared__ __attribute__((aligned(1024))) uint8_t smem[ROW_KS * D * SLOT];
    const int lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4;
    const int ks = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    // rows that are read together lie in other banks: 4 neighbouring chunks of each of 4 rows, one of each of 16
    auto swz = [](int row) { return XC == 1 ? 4 * row : row; };
    uint8_t* mine = smem + ks * D * SLOT;
    const int64_t total = (int64_t)count_tiles<BM>(p) * ntiles;
    const int steps = p.KT > ks ? (p.KT - ks - 1) / ROW_KS + 1 : 0;
    for (int64_t tile = blockIdx.x; tile < total; tile += gridDim.x) {
        int e, nrows;
        int64_t row0;
        const int mt = (int)(tile / ntiles), nt = (int)(tile - (int64_t)mt * ntiles);
        find_tile<BM>(p, mt, e, row0, nrows);
        // Copy i fills rows 4 i .. 4 i + 3; lane l takes row l / 16, position l %
        // 16, which holds chunk (l % 16) ^ swz(row). Rows past the tile repeat its
        // last one; an id that is no row reads row 0, and is not used.
        const uint8_t* x[XC];
        int chunk[XC];
#pragma unroll
        for (int i = 0; i < XC; ++i) {
            const int row = 4 * i + g;
            const int64_t from = max(source_row(p, row0 + min(row, nrows - 1)), (int64_t)0);
            chunk[i] = (r ^ swz(row)) * 8;
            x[i] = (const uint8_t*)p.x + from * p.x_stride * 2;
        }
        const uint8_t* w = p.w + e * p.w_expert + (int64_t)nt * p.KT * 1024 + lane * 16;
        // dword l of the scales: two or one of channel and group; lanes past them repeat the last
        constexpr int PER = 4 / (int)sizeof(ST), SL = 16 / PER;
        const int sg = min(lane / SL, G - 1);
        const ST* scale = (const ST*)p.scale + e * p.scale_expert + nt * 16 + lane % SL * PER;
        const int last_group = (p.K - 1) >> p.group_shift;
        auto issue = [&](int i) __attribute__((always_inline)) {
            const int kt = i * ROW_KS + ks;
            uint8_t* to = mine + i % D * SLOT;
            g2l16(w + (int64_t)kt * 1024, to);
#pragma unroll
            for (int c = 0; c < XC; ++c)  // past K: any value, cut below
                g2l16(x[c] + (int64_t)min(kt * 128 + chunk[c], p.K - 8) * 2, to + X + c * 1024);
            const int row = min(G == 1 ? (kt * 128) >> p.group_shift : kt * G + sg, last_group);
            g2l4(scale + (int64_t)row * p.Np, to + S);
        };
        v4f acc = {0.f, 0.f, 0.f, 0.f};
        for (int i = 0; i < D - 1 && i < steps; ++i) issue(i);
        const int row = r % BM;  // rows that are none: any of them
        for (int i = 0; i < steps; ++i) {
            if (i + D - 1 < steps) issue(i + D - 1);
            wait_steps<LD, D - 1>(steps - 1 - i);
            const uint8_t* at = mine + i % D * SLOT;
            const v4u d = *reinterpret_cast<const v4u*>(at + lane * 16);
            frag f[4];
            const int left = p.K - (i * ROW_KS + ks) * 128;
#pragma unroll
            for (int k = 0; k < 4; ++k)
                f[k] = *reinterpret_cast<const frag*>(at + X + row * 256 + ((4 * k + g) ^ swz(row)) * 16);
            if (left < 128) {
#pragma unroll
                for (int k = 0; k < 4; ++k)
                    if (32 * k + 8 * g >= left) f[k] = __builtin_bit_cast(frag, (v4u){0, 0, 0, 0});
            }
#pragma unroll
            for (int j = 0; j < G; ++j) {
                const s4 s = *reinterpret_cast<const s4*>(at + S + (j * 16 + 4 * g) * sizeof(ST));
                v4f t = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int k = j * GS; k < j * GS + GS; ++k) t = Op::mfma(Op::weights(d[k]), f[k], t);
#pragma unroll
                for (int v = 0; v < 4; ++v) acc[v] = fmaf((float)s[v], t[v], acc[v]);
            }
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // this slot has been read: the next copy may fill it
        }
        __syncthreads();
        v4f* sums = reinterpret_cast<v4f*>(smem);
        sums[ks * 64 + lane] = acc;
        __syncthreads();
        if (threadIdx.x < 64) {
#pragma unroll
            for (int k = 1; k < ROW_KS; ++k) acc += sums[k * 64 + lane];
            if (r < nrows) store_sums<Op>(p, row0 + r, nt * 16 + 4 * g, vec, acc);
        }
        __syncthreads();
    }
    zero_rest_any(p, vec);
}

template <int XC, int D>
hipError_t launch_row(const Int4Call& p, int x_dtype, int scale_dtype, bool vec, hipStream_t s) {
    return by_int4_types(x_dtype, scale_dtype, 1 << p.group_shift, [&](auto x, auto sc, auto gs) {
        const int ntiles = p.Np / 16;
        const int64_t tiles = max_tiles(p.rows, 4 * XC, p.E) * ntiles;
        hipLaunchKernelGGL((int4_row_kernel<decltype(x), decltype(sc), decltype(gs)::value, XC, D>),
                           dim3((unsigned)(tiles < 4096 ? tiles : 4096)), dim3(64 * ROW_KS), 0, s, p, ntiles, (int)vec);
        return hipGetLastError();
    });
}

hipError_t launch_int4_row(const Int4Call& p, int x_dtype, int scale_dtype, Int4Tile tile, bool vec, hipStream_t s) {
    if (tile == Int4Tile::T16x16) return launch_row<4, 3>(p, x_dtype, scale_dtype, vec, s);
    // one to a CU with all its loads on their way, or two
    return max_tiles(p.rows, 4, p.E) * (p.Np / 16) <= 256 ? launch_row<1, 8>(p, x_dtype, scale_dtype, vec, s)
                                                          : launch_row<1, 4>(p, x_dtype, scale_dtype, vec, s);
}

}  // namespace miexp
