// Products of many rows with 4-bit weights, in tiles of 256 rows x 192 channels (or
// 128): one workgroup per CU, its eight waves in two groups that share the SIMDs, a
// wave of each group to one, and take turns at making weights.
//
// A step is 128 values of K. A wave multiplies 128 rows by 48 channels (32 with
// groups of less than 128): first it makes 16 bits of its channels' weights in
// registers, then it goes over its eight row tiles. That is two phases: A, the
// weights and two row tiles, and B, the other six; a barrier ends each, and group
// 1 runs one behind group 0. So while one wave of a SIMD makes weights (3 x 52
// instructions for bfloat16, as long as three or four row tiles take) the other
// one multiplies, and then both do. Row tiles of 16 go to the groups in turn, so
// that a tile with few rows keeps both busy.
//
// Copies into LDS (two stages): a group's rows by its own waves, the ones that
// phase A reads (low) and those of phase B (high); weights and scales by group 0.
// Of step t, phase A issues the weights of t + 1, and phase B high of t + 1, one
// beside each row tile, and low of t + 2: each into what has been read before. So
// the copies have two phases at least to arrive; at the end of a phase the next
// one's are waited for.
//
// 8192 x 4096 x 7168 430 to 450 us (1.07 to 1.12 PFLOP/s; the library's product of
// bfloat16 weights 372), in groups of 64 470 to 500, of 32 590 to 603; 8192 rows of
// 32 experts of 7168 x 2048 300 to 325. Where the first took 446, 392 without the
// copies, 408 without making weights, 421 without storing results: no one part
// holds it; 704 tiles are two and three quarters rounds of the CUs. Before: all
// eight row tiles behind the weights in one phase 500, four in each phase 486, the
// copies of a step all at its start 472, stores of four channels 446.
#include "int4_common.hpp"
#include "lds_copy.hpp"

namespace miexp {

using mimoe::g2l16s;
using mimoe::g2l4s;

namespace wide4 {
constexpr int MT = 8, WN = 4, BM = 256;
constexpr int ML = 2;                                        // row tiles of phase A
constexpr int X_GROUP = BM / 2 * 256, X = 2 * X_GROUP;       // bytes of rows
constexpr int XC = X_GROUP / 1024 / WN, LOW = XC * ML / MT;  // copies of a wave: of its group's rows, of those of A
template <class ST, int GS>
struct Shape {
    // With groups of 32 and 64 a wave has 32 channels: 48, their scales and the
    // sums do not fit its 256 registers, and scaling bounds these anyway.
    static constexpr int NT = GS == 4 ? 3 : 2, BN = 16 * NT * WN;
    static constexpr int G = 4 / GS, W = BN * 64, S = (G * BN * (int)sizeof(ST) + 255) / 256 * 256;
    static constexpr int STAGE = X + W + S;
    static constexpr int WC = NT + (S / 256 + WN - 1) / WN;  // copies of a wave: weights and scales
    static_assert(2 * STAGE <= 160 * 1024, "LDS budget");
};
// Rows of each of `tiles` tiles that share `rows` evenly, in 32s: at most BM,
// as there are ceil(rows / BM). Up to 2^31 - 1 rows, so nothing is added to them
// before the division.
constexpr int tile_height(int rows, int tiles) { return ((rows - 1) / tiles + 32) / 32 * 32; }
static_assert(tile_height(1, 1) == 32 && tile_height(256, 1) == 256 && tile_height(257, 2) == 160 &&
                  tile_height(270, 2) == 160 && tile_height(2147483392, 8388607) == BM,
              "all rows in tiles of at most BM");
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

// Results of 16 bits, 16 bytes of a lane at a time: of two tiles of 16 x 16, lanes
// of odd rows of 16 take the second one's and give the first one's, so that each
// has eight neighbouring channels. For destinations aligned to that. (Four channels
// of a lane: 6 to 9 % of the call were its stores.)
template <class T, class Op, int GROUP, int NT>
__device__ __forceinline__ void store_pairs(const Int4Call& p, int64_t row0, int nrows, int n0,
                                            const v4f (&acc)[wide4::MT][NT]) {
    const int lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4;
    typedef T t4 __attribute__((ext_vector_type(4)));
    typedef unsigned v2u __attribute__((ext_vector_type(2)));
    auto packed = [&](int m, int n) __attribute__((always_inline)) {
        float y[4];
        finish_sums<Op>(p, row0 + min(32 * m + 16 * GROUP + r, nrows - 1), n0 + n * 16 + 4 * g, acc[m][n], y);
        return __builtin_bit_cast(v2u, (t4){(T)y[0], (T)y[1], (T)y[2], (T)y[3]});
    };
    auto pair = [&](int ma, int na, int mb, int nb) __attribute__((always_inline)) {
        if (32 * ma + 16 * GROUP >= nrows) return;  // mb >= ma
        const v2u a = packed(ma, na), b = packed(mb, nb);
        const auto lo = __builtin_amdgcn_permlane16_swap(a[0], b[0], false, false);
        const auto hi = __builtin_amdgcn_permlane16_swap(a[1], b[1], false, false);
        const v4u v = {lo[0], hi[0], lo[1], hi[1]};
        const bool second = g & 1;
        const int row = 32 * (second ? mb : ma) + 16 * GROUP + r, n = n0 + (second ? nb : na) * 16 + 8 * (g >> 1);
        if (row >= nrows || n >= p.N) return;
        T* to = reinterpret_cast<T*>(p.out) + (row0 + row) * p.out_stride + n;
        if (n + 8 <= p.N) {
            *reinterpret_cast<v4u*>(to) = v;
        } else {
            typedef T t8 __attribute__((ext_vector_type(8)));
            const t8 x = __builtin_bit_cast(t8, v);
#pragma unroll
            for (int e = 0; e < 8; ++e)
                if (n + e < p.N) to[e] = x[e];
        }
    };
#pragma unroll
    for (int m = 0; m < wide4::MT; ++m) {
        pair(m, 0, m, 1);
        if constexpr (NT == 3) {
            if (m % 2 == 0) pair(m, 2, m + 1, 2);
        }
    }
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

    // A copy fills four rows of the group; lane l takes row l / 16, position l %
    // 16. Group row j is row 32 (j / 16) + 16 GROUP + j % 16 of the tile; rows past
    // the tile repeat its last one.
    const uint8_t* x_base = (const uint8_t*)p.x + (p.row_ids ? 0 : row0 * p.x_stride * 2);
    uint32_t x_off[XC];
    const int chunk_of_lane = lane & 15;
    auto group_row = [&](int i) __attribute__((always_inline)) {
        return 4 * (i < LOW ? wn * LOW + i : WN * LOW + wn * (XC - LOW) + i - LOW);
    };
#pragma unroll
    for (int i = 0; i < XC; ++i) {
        const int j = group_row(i) + (lane >> 4);
        const int m = min(32 * (j >> 4) + 16 * GROUP + (j & 15), nrows - 1);
        const int64_t from = p.row_ids ? max(source_row(p, row0 + m), (int64_t)0) : m;
        x_off[i] = (uint32_t)(from * p.x_stride) * 2 + (chunk_of_lane ^ (j & 15)) * 16;
    }
    // past K, in a last step that K ends in: the step's first chunk
    auto cut = [&](int i) __attribute__((always_inline)) {
        const int chunk = chunk_of_lane ^ ((group_row(i) + (lane >> 4)) & 15);
        return (uint32_t)(chunk * 8 >= rest ? chunk * 16 : 0);
    };
    auto issue_row = [&](int kb, int i) __attribute__((always_inline)) {
        const uint32_t off = x_off[i] - (kb == p.KT - 1 && rest != 128 ? cut(i) : 0);
        g2l16s(x_base + (int64_t)kb * 256, off, smem + (kb & 1) * Z::STAGE + GROUP * X_GROUP + group_row(i) * 256);
    };
    auto issue_low = [&](int kb) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < LOW; ++i) issue_row(kb, i);
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
        for (int i = 0; i < Z::WC - NT; ++i) {
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
    // The compiler would sink each LDS read to its use and wait there for it: what
    // a fence of the scheduler parts stays in this order.
    auto fence = [] { __builtin_amdgcn_sched_barrier(0); };
    frag x[2][4];
    auto fragments = [&](int m, int kb, auto last_c) __attribute__((always_inline)) {
        const uint8_t* rows = smem + (kb & 1) * Z::STAGE + GROUP * X_GROUP + (m * 16 + r) * 256;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            x[m & 1][i] = *reinterpret_cast<const frag*>(rows + ((4 * i + g) ^ r) * 16);
            if (decltype(last_c)::value && 32 * i + 8 * g >= rest) x[m & 1][i] = __builtin_bit_cast(frag, (v4u){0, 0, 0, 0});
        }
    };
    auto make_weights = [&](int kb, auto last_c) __attribute__((always_inline)) {
        const uint8_t* sw = smem + (kb & 1) * Z::STAGE + X + wn * NT * 1024;
        const uint8_t* ss = smem + (kb & 1) * Z::STAGE + X + W + wn * NT * 16 * sizeof(ST);
        v4u d[NT];
        s4 s[NT][G];
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            d[n] = *reinterpret_cast<const v4u*>(sw + n * 1024 + lane * 16);
#pragma unroll
            for (int j = 0; j < G; ++j) s[n][j] = *reinterpret_cast<const s4*>(ss + (j * BN + n * 16 + 4 * g) * sizeof(ST));
        }
        fragments(0, kb, last_c);
        fence();
#pragma unroll
        for (int n = 0; n < NT; ++n) {
#pragma unroll
            for (int i = 0; i < 4; ++i) w[n][i] = Op::weights(d[n][i]);
#pragma unroll
            for (int j = 0; j < G; ++j)
#pragma unroll
                for (int v = 0; v < 4; ++v) scale[n][j][v] = (float)s[n][j][v];
        }
    };
    // The row tiles of a phase; the fragments of each are read while the one
    // before is multiplied. MORE: a copy of the next step's high rows goes out
    // beside each.
    auto multiply = [&](int kb, auto high, auto more, auto last_c) __attribute__((always_inline)) {
        constexpr int FROM = decltype(high)::value ? ML : 0, TO = decltype(high)::value ? MT : ML;
#pragma unroll
        for (int m = FROM; m < TO; ++m) {
            fence();
            if (m + 1 < TO) fragments(m + 1, kb, last_c);
            if constexpr (decltype(more)::value) issue_row(kb + 1, LOW + m - FROM);
            fence();
            if (32 * m + 16 * GROUP < nrows) {
#pragma unroll
                for (int j = 0; j < G; ++j)
#pragma unroll
                    for (int n = 0; n < NT; ++n) {
                        v4f t = (v4f){0.f, 0.f, 0.f, 0.f};
#pragma unroll
                        for (int i = j * GS; i < j * GS + GS; ++i) t = Op::mfma(w[n][i], x[m & 1][i], t);
#pragma unroll
                        for (int v = 0; v < 4; ++v) acc[m][n][v] = fmaf(scale[n][j][v], t[v], acc[m][n][v]);
                    }
            }
        }
        fence();
    };
    static_assert(XC - LOW == MT - ML, "a copy for each row tile of phase B");
    // two more steps follow, one, or none
    auto step = [&](int t, auto more2, auto more1) __attribute__((always_inline)) {
        constexpr bool M2 = decltype(more2)::value, M1 = decltype(more1)::value;
        typedef IntC<!M1> Last;
        // A
        make_weights(t, Last{});
        if constexpr (M1 && GROUP == 0) issue_weights(t + 1);
        multiply(t, IntC<0>{}, IntC<0>{}, Last{});
        // high of this step is there: later are low of t + 1 and what this phase issued
        phase_end<M1 ? LOW + (GROUP == 0 ? Z::WC : 0) : 0>();
        // B
        fragments(ML, t, Last{});
        multiply(t, IntC<1>{}, more1, Last{});
        if constexpr (M2) issue_low(t + 2);
        // low and weights of t + 1 are there: later are its high and low of t + 2
        phase_end<(M1 ? XC - LOW : 0) + (M2 ? LOW : 0)>();
    };
    if constexpr (GROUP == 0) issue_weights(0);
    issue_low(0);
#pragma unroll
    for (int i = LOW; i < XC; ++i) issue_row(0, i);
    if (p.KT > 1) {
        issue_low(1);
        phase_end<XC>();
    } else {
        phase_end<XC - LOW>();
    }
    if constexpr (GROUP == 1) phase_end();
    for (int t = 0; t < p.KT - 2; ++t) step(t, IntC<1>{}, IntC<1>{});
    if (p.KT > 1) step(p.KT - 2, IntC<0>{}, IntC<1>{});
    step(p.KT - 1, IntC<0>{}, IntC<0>{});
    if constexpr (GROUP == 0) phase_end();
    if (vec && p.out_dtype != MI_LAYER_F32) {
        if (p.out_dtype == MI_LAYER_F16)
            store_pairs<_Float16, Op, GROUP, NT>(p, row0, nrows, n0 + wn * NT * 16, acc);
        else
            store_pairs<__bf16, Op, GROUP, NT>(p, row0, nrows, n0 + wn * NT * 16, acc);
        return;
    }
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
    if (!is_for_rows(p)) return;
    Tiles tile;
    const int mt = blockIdx.x / ntiles, nt = blockIdx.x % ntiles;
    if (find_expert<BM>(p, mt, tile)) {
        // an expert's rows in tiles of the same height: 270 rows cost less as 135 twice than as 256 and 14
        const int rows = tile.end - tile.row, height = wide4::tile_height(rows, tile.tiles);
        const int from = (mt - tile.first) * height, nrows = min(height, rows - from);
        if (nrows > 0) {
            if (threadIdx.x < 256)
                wide_run<XT, ST, GS, 0>(p, smem, tile.e, (int64_t)tile.row + from, nrows, nt * BN, vec);
            else
                wide_run<XT, ST, GS, 1>(p, smem, tile.e, (int64_t)tile.row + from, nrows, nt * BN, vec);
        }
    }
    zero_rest_any(p, vec);
}

hipError_t launch_int4_wide(const Int4Call& p, int x_dtype, int scale_dtype, hipStream_t s) {
    const int per16 = p.out_dtype == MI_LAYER_F32 ? 4 : 8;
    const bool vec = (uint64_t)p.out % 16 == 0 && p.out_stride % per16 == 0;
    return by_int4_types(x_dtype, scale_dtype, 1 << p.group_shift, [&](auto x, auto sc, auto gs) {
        constexpr int BN = wide4::Shape<decltype(sc), decltype(gs)::value>::BN;
        const int64_t nt = (p.N + BN - 1) / BN, tiles = max_tiles(p.rows, wide4::BM, p.E) * nt;
        hipLaunchKernelGGL((int4_wide_kernel<decltype(x), decltype(sc), decltype(gs)::value>), dim3((unsigned)tiles),
                           dim3(512), 0, s, p, (int)nt, (int)vec);
        return hipGetLastError();
    });
}

}  // namespace miexp
