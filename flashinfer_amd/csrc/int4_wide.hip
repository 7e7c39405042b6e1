// Products of many rows with 4-bit weights, in tiles of 256 rows x 192 channels (or
// 128): one workgroup per CU, its eight waves in two groups that share the SIMDs, a
// wave of each group to one, and take turns at making weights.
//
// A step is 128 values of K. A wave multiplies 128 rows by 48 channels (32 with
// groups of less than 128): first it
// makes 16 bits of its channels' weights in registers, then it goes over its
// eight row tiles. That is two phases: A, the weights and row tiles 0 - 3, and B,
// row tiles 4 - 7; a barrier ends each, and group 1 runs one behind group 0. So
// while one wave of a SIMD makes weights (3 x 52 instructions for bfloat16) the
// other one multiplies. Row tiles of 16 go to the groups in turn, so that a tile
// with few rows keeps both busy.
//
// Copies into LDS (two stages): a group's rows in halves, the ones that phase A
// reads (low) and those of phase B (high), by its own waves; weights and scales
// by group 0. Of step t, phase A issues high and the weights of t + 1 and phase B
// low of t + 2, into what the phase before has read, so that rows have three
// phases to arrive and weights two. All but what phase B issued has to be there
// when it ends: that is what the next step reads.
#include "int4_common.hpp"
#include "lds_copy.hpp"

namespace miexp {

using mimoe::g2l16s;
using mimoe::g2l4s;

namespace wide4 {
constexpr int MT = 8, WN = 4, BM = 256;
constexpr int X_HALF = 64 * 256, X = 4 * X_HALF;  // bytes of rows: [group][low, high]
constexpr int LOW = X_HALF / 1024 / WN;           // copies of a wave for half of its group's rows
template <class ST, int GS>
struct Shape {
    // With groups of 32 and 64 a wave has 32 channels: 48, their scales and the
    // sums do not fit its 256 registers, and scaling bounds these anyway.
    static constexpr int NT = GS == 4 ? 3 : 2, BN = 16 * NT * WN;
    static constexpr int G = 4 / GS, W = BN * 64, S = (G * BN * (int)sizeof(ST) + 255) / 256 * 256;
    static constexpr int STAGE = X + W + S;
    static_assert(2 * STAGE <= 160 * 1024, "LDS budget");
};
}  // namespace wide4

// End of a phase: this wave's LDS reads are done and at most N of its copies
// are in flight; then the workgroup's barrier.
template <int N>
__device__ __forceinline__ void phase_end() {
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(N) : "memory");
}
__device__ __forceinline__ void phase_end() {
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
}

template <class XT, class ST, int GS, int GROUP>
__device__ __forceinline__ void wide_run(const Int4Call& p, uint8_t* smem, int e, int64_t row0, int nrows, int n0,
                                         bool vec) {
    using namespace wide4;
    typedef Shape<ST, GS> Z;
    typedef Operand<XT> Op;
    typedef typename Op::frag frag;
    typedef ST s4 __attribute__((ext_vector_type(4)));
    constexpr int G = Z::G, NT = Z::NT, BN = Z::BN, W = Z::W;
    const int lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4;
    const int wn = __builtin_amdgcn_readfirstlane((threadIdx.x >> 6) & 3);
    const int rest = p.K - (p.KT - 1) * 128;  // values of the last step: 8 .. 128

    // Copy i of a half fills rows 4 (wn LOW + i) .. + 3 of its 64; lane l takes
    // row l / 16, position l % 16. Group row j is row 32 (j / 16) + 16 GROUP + j %
    // 16 of the tile; rows past the tile repeat its last one.
    const uint8_t* x_base = (const uint8_t*)p.x + (p.row_ids ? 0 : row0 * p.x_stride * 2);
    uint32_t x_off[2][LOW];
    const int chunk_of_lane = lane & 15;
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int i = 0; i < LOW; ++i) {
            const int j = h * 64 + 4 * (wn * LOW + i) + (lane >> 4);
            const int m = min(32 * (j >> 4) + 16 * GROUP + (j & 15), nrows - 1);
            const int64_t from = p.row_ids ? max(source_row(p, row0 + m), (int64_t)0) : m;
            x_off[h][i] = (uint32_t)(from * p.x_stride) * 2 + (chunk_of_lane ^ (j & 15)) * 16;
        }
    // past K, in a last step that K ends in: the step's first chunk
    auto cut = [&](int i) __attribute__((always_inline)) {
        const int chunk = chunk_of_lane ^ ((4 * (wn * LOW + i) + (lane >> 4)) & 15);
        return (uint32_t)(chunk * 8 >= rest ? chunk * 16 : 0);
    };
    auto issue_rows = [&](int kb, int h) __attribute__((always_inline)) {
        uint8_t* to = smem + (kb & 1) * Z::STAGE + (GROUP * 2 + h) * X_HALF + wn * LOW * 1024;
        const uint8_t* x = x_base + (int64_t)kb * 256;
        if (kb == p.KT - 1 && rest != 128) {
#pragma unroll
            for (int i = 0; i < LOW; ++i) g2l16s(x, x_off[h][i] - cut(i), to + i * 1024);
        } else {
#pragma unroll
            for (int i = 0; i < LOW; ++i) g2l16s(x, x_off[h][i], to + i * 1024);
        }
    };
    const uint8_t* w_base = p.w + e * p.w_expert;
    const int last_tile = p.Np / 16 - 1;
    constexpr int D = BN * (int)sizeof(ST) / 4;  // dwords of a group's scales
    const uint8_t* s_base = (const uint8_t*)p.scale + (e * p.scale_expert + n0) * (int64_t)sizeof(ST);
    const int row_bytes = p.Np * (int)sizeof(ST), last_group = (p.K - 1) >> p.group_shift;
    auto issue_weights = [&](int kb) __attribute__((always_inline)) {
        uint8_t* to = smem + (kb & 1) * Z::STAGE + X;
#pragma unroll
        for (int i = 0; i < NT; ++i) {
            const int t = wn * NT + i;
            g2l16s(w_base + ((int64_t)min(n0 / 16 + t, last_tile) * p.KT + kb) * 1024, lane * 16, to + t * 1024);
        }
#pragma unroll
        for (int i = 0; i < (Z::S / 256 + WN - 1) / WN; ++i) {
            const int c = (wn + i * WN) % (Z::S / 256), d = c * 64 + lane;
            const int row = min(G == 1 ? (kb * 128) >> p.group_shift : kb * G + d / D, last_group);
            g2l4s(s_base, (uint32_t)row * row_bytes + min(d % D * 4, row_bytes - n0 * (int)sizeof(ST) - 4),
                  to + W + c * 256);
        }
    };

    v4f acc[MT][NT];
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int n = 0; n < NT; ++n) acc[m][n] = (v4f){0.f, 0.f, 0.f, 0.f};
    frag w[NT][4];
    v4f scale[NT][G];
    auto make_weights = [&](int kb) __attribute__((always_inline)) {
        const uint8_t* sw = smem + (kb & 1) * Z::STAGE + X + wn * NT * 1024;
        const uint8_t* ss = smem + (kb & 1) * Z::STAGE + X + W + wn * NT * 16 * sizeof(ST);
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            const v4u d = *reinterpret_cast<const v4u*>(sw + n * 1024 + lane * 16);
#pragma unroll
            for (int i = 0; i < 4; ++i) w[n][i] = Op::weights(d[i]);
#pragma unroll
            for (int j = 0; j < G; ++j) {
                const s4 s = *reinterpret_cast<const s4*>(ss + (j * BN + n * 16 + 4 * g) * sizeof(ST));
#pragma unroll
                for (int v = 0; v < 4; ++v) scale[n][j][v] = (float)s[v];
            }
        }
    };
    // Row tiles go one by one: a branch each, which also keeps the compiler from
    // spreading the sums of several over more registers than there are.
    auto fragments = [&](frag (&x)[4], const uint8_t* rows, auto last_c) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            x[i] = *reinterpret_cast<const frag*>(rows + r * 256 + ((4 * i + g) ^ r) * 16);
            if (decltype(last_c)::value && 32 * i + 8 * g >= rest) x[i] = __builtin_bit_cast(frag, (v4u){0, 0, 0, 0});
        }
    };
    auto multiply = [&](int kb, auto half, auto last_c) __attribute__((always_inline)) {
        constexpr int H = decltype(half)::value;
        const uint8_t* sx = smem + (kb & 1) * Z::STAGE + (GROUP * 2 + H) * X_HALF;
        frag x[2][4];
        fragments(x[0], sx, last_c);
#pragma unroll
        for (int m = 0; m < 4; ++m) {
            if (32 * (H * 4 + m) + 16 * GROUP >= nrows) break;
            if (m < 3) fragments(x[(m + 1) & 1], sx + (m + 1) * 4096, last_c);
#pragma unroll
            for (int j = 0; j < G; ++j) {
                v4f t[NT];
#pragma unroll
                for (int n = 0; n < NT; ++n) t[n] = (v4f){0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int i = j * GS; i < j * GS + GS; ++i)
#pragma unroll
                    for (int n = 0; n < NT; ++n) t[n] = Op::mfma(w[n][i], x[m & 1][i], t[n]);
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int v = 0; v < 4; ++v)
                        acc[H * 4 + m][n][v] = fmaf(scale[n][j][v], t[n][v], acc[H * 4 + m][n][v]);
            }
        }
    };
    auto step = [&](int t, auto last_c) __attribute__((always_inline)) {
        // A
        if (t + 1 < p.KT) {
            issue_rows(t + 1, 1);
            if constexpr (GROUP == 0) issue_weights(t + 1);
        }
        make_weights(t);
        multiply(t, IntC<0>{}, last_c);
        __builtin_amdgcn_sched_barrier(0);
        phase_end();
        // B
        if (t + 2 < p.KT) issue_rows(t + 2, 0);
        multiply(t, IntC<1>{}, last_c);
        __builtin_amdgcn_sched_barrier(0);
        if (t + 2 < p.KT)
            phase_end<LOW>();
        else
            phase_end<0>();
    };
    if constexpr (GROUP == 0) issue_weights(0);
    issue_rows(0, 0);
    issue_rows(0, 1);
    if (p.KT > 1) {
        issue_rows(1, 0);
        phase_end<LOW>();
    } else {
        phase_end<0>();
    }
    if constexpr (GROUP == 1) phase_end();
    for (int t = 0; t < p.KT - 1; ++t) step(t, IntC<0>{});
    step(p.KT - 1, IntC<1>{});
    if constexpr (GROUP == 0) phase_end();
#pragma unroll
    for (int m = 0; m < MT; ++m) {
        const int row = 32 * m + 16 * GROUP + r;
        if (row >= nrows) continue;
#pragma unroll
        for (int n = 0; n < NT; ++n) store_sums<Op>(p, row0 + row, n0 + (wn * NT + n) * 16 + 4 * g, vec, acc[m][n]);
    }
}

template <class XT, class ST, int GS>
__global__ __launch_bounds__(512, 2) void int4_wide_kernel(Int4Call p, int ntiles, int vec) {
    using namespace wide4;
    constexpr int BN = Shape<ST, GS>::BN;
    __shared__ __attribute__((aligned(1024))) uint8_t smem[2 * Shape<ST, GS>::STAGE];
    Tiles tile;
    const int mt = blockIdx.x / ntiles, n0 = (int)(blockIdx.x % ntiles) * BN;
    if (!find_expert<BM>(p, mt, tile)) return zero_rest_any(p, vec);
    const int64_t row0 = (int64_t)tile.row + (int64_t)(mt - tile.first) * BM;
    const int nrows = (int)min((int64_t)BM, tile.end - row0);
    if (threadIdx.x < 256)
        wide_run<XT, ST, GS, 0>(p, smem, tile.e, row0, nrows, n0, vec);
    else
        wide_run<XT, ST, GS, 1>(p, smem, tile.e, row0, nrows, n0, vec);
    zero_rest_any(p, vec);
}

hipError_t launch_int4_wide(const Int4Call& p, int x_dtype, int scale_dtype, bool vec, hipStream_t s) {
    return by_int4_types(x_dtype, scale_dtype, 1 << p.group_shift, [&](auto x, auto sc, auto gs) {
        constexpr int BN = wide4::Shape<decltype(sc), decltype(gs)::value>::BN;
        const int64_t nt = (p.N + BN - 1) / BN, tiles = max_tiles(p.rows, wide4::BM, p.E) * nt;
        hipLaunchKernelGGL((int4_wide_kernel<decltype(x), decltype(sc), decltype(gs)::value>), dim3((unsigned)tiles),
                           dim3(512), 0, s, p, (int)nt, (int)vec);
        return hipGetLastError();
    });
}

}  // namespace miexp
