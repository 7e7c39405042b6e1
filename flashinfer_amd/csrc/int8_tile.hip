// Integer products of some rows: BM x BN tiles staged through LDS, with K shared
// by groups of waves.
//
// KS groups of four waves each take every KS-th step of 128 bytes of K. A
// group copies its rows of both operands global -> LDS into one of STAGES
// buffers, STAGES - 1 of its steps ahead; the groups share one barrier a turn.
// What a small tile costs is the length of that chain (wait, barrier, LDS
// reads, a few MFMAs), so sharing K shortens it and gives each SIMD a wave to
// run while another one waits. The groups' integer sums meet in LDS at the end.
// Against N = 4096, K = 7168 (29 MB of weights, 6 us at 5 TB/s): M = 1 and 64
// 8.3 and 8.9 us with 32 x 32 tiles and K in four (64 x 64 with K in two 14 and
// 15, whole 17), 128 11.8 (32 x 64, four), 256 16.7 (64 x 64, two; 18.8 whole),
// 512 23.8 (64 x 128, two; 26.2 whole), 1024 35.9 (128 x 128, two; 40.4 whole),
// 2048 59 (128 x 128 whole, two workgroups to a CU, 2.0 POP/s).
//
// LDS rows are 128 bytes, 16-byte chunk c of row r at position c ^ swzq(r).
// Copies past K read zeros; rows past the tile repeat its last one and are not
// stored.
#include "int8_common.hpp"

namespace miexp {

using mimoe::g2l16s;
using mimoe::g2l16s_once;
using mimoe::swzq;

template <int N>
__device__ __forceinline__ void wait_copies() {
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}

// ONCE: the weights pass the caches by.
template <class T, int BM, int BN, int STAGES, int KS, bool ONCE>
__device__ __forceinline__ void tile_run(const Int8Call& p, uint8_t* smem, int e, int64_t row0, int nrows, int n0,
                                         bool vec) {
    constexpr int MT = BM / 32, NT = BN / 32;  // 16 x 16 tiles of a wave
    constexpr int A_LD = BM / 32, B_LD = BN / 32, LD = A_LD + B_LD;  // 1 KB copies of a wave
    constexpr int STAGE = (BM + BN) * 128;
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane((threadIdx.x >> 6) & 3);
    const int ks = __builtin_amdgcn_readfirstlane(threadIdx.x >> 8);
    const int r = lane & 15, g = lane >> 4;
    const int wm = wave & 1, wn = wave >> 1;
    const int KB = (p.K + 127) / 128;
    const int rest = p.K - (KB - 1) * 128;  // bytes of the last step: 16 .. 128

    // Loader: copy i of a wave fills 8 LDS rows; lane l takes row l / 8, position
    // l % 8. Its source is a base in SGPRs (the tile's first row; a itself with
    // row_ids) and a 32-bit offset. An id that is no row reads row 0: its scale
    // is NaN.
    const int8_t* a_base = p.a + (p.row_ids ? 0 : row0 * p.a_stride);
    const int8_t* b_base = p.b + e * p.b_expert_stride + (int64_t)n0 * p.b_stride;
    auto lds_row = [&](int i) __attribute__((always_inline)) {
        return 8 * (i < A_LD ? wave * A_LD + i : wave * B_LD + i - A_LD) + (lane >> 3);
    };
    auto chunk = [&](int i) __attribute__((always_inline)) { return ((lane & 7) ^ swzq(lds_row(i))) * 16; };
    uint32_t off[LD];
#pragma unroll
    for (int i = 0; i < LD; ++i) {
        const int row = lds_row(i);
        if (i < A_LD) {
            const int m = min(row, nrows - 1);
            const int64_t from = p.row_ids ? max(source_row(p, row0 + m), (int64_t)0) : m;
            off[i] = (uint32_t)(from * p.a_stride) + chunk(i);
        } else {
            off[i] = (uint32_t)(min(row, p.N - 1 - n0) * p.b_stride) + chunk(i);
        }
    }
    // In a last step that K ends in, lanes past K read the step's first chunk
    // (branch-free: a branch here would part the copies from the LDS reads they
    // overlap with), and the fragments are cut to zeros.
    uint32_t cut[LD];
#pragma unroll
    for (int i = 0; i < LD; ++i) cut[i] = chunk(i) >= rest ? chunk(i) : 0;
    uint8_t* mine = smem + ks * STAGES * STAGE;
    auto issue = [&](int kb, int stage) __attribute__((always_inline)) {
        uint8_t* s = mine + stage * STAGE;
        const int8_t *a = a_base + kb * 128, *b = b_base + kb * 128;
        const uint32_t last = kb == KB - 1 ? ~0u : 0u;
#pragma unroll
        for (int i = 0; i < LD; ++i)
            if (i < A_LD)
                g2l16s(a, off[i] - (cut[i] & last), s + (wave * A_LD + i) * 1024);
            else if (ONCE)
                g2l16s_once(b, off[i] - (cut[i] & last), s + (BM / 8 + wave * B_LD + i - A_LD) * 1024);
            else
                g2l16s(b, off[i] - (cut[i] & last), s + (BM / 8 + wave * B_LD + i - A_LD) * 1024);
    };
    Scales<MT, NT> scales;
    scales.load(p, e, row0, nrows, wm * (BM / 2), n0 + wn * (BN / 2));
    v4i acc[MT][NT];
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int n = 0; n < NT; ++n) acc[m][n] = (v4i){0, 0, 0, 0};
    // turn t: step t * KS + ks of K, in buffer t % STAGES
    const int turns = (KB + KS - 1) / KS, steps = KB > ks ? (KB - ks - 1) / KS + 1 : 0;  // of this group
#pragma unroll
    for (int t = 0; t < STAGES - 1; ++t)
        if (t < steps) issue(t * KS + ks, t);
    int cur = 0;
    auto turn = [&](int t, auto last_c) __attribute__((always_inline)) {
        // the copies of turn t are the oldest; those of STAGES - 2 later ones may be in flight
        if (t + STAGES - 2 < steps)
            wait_copies<LD*(STAGES - 2)>();
        else
            wait_copies<0>();
        __syncthreads();
        const int next = cur == 0 ? STAGES - 1 : cur - 1;  // buffer of turn t - 1: of t + STAGES - 1
        if (t + STAGES - 1 < steps) issue((t + STAGES - 1) * KS + ks, next);
        const uint8_t* sA = mine + cur * STAGE + wm * (BM / 2) * 128;
        const uint8_t* sB = mine + cur * STAGE + BM * 128 + wn * (BN / 2) * 128;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int at = r * 128 + (((h * 4 + g) ^ swzq(r)) << 4);
            v4i fa[MT], fb[NT];
#pragma unroll
            for (int n = 0; n < NT; ++n) fb[n] = *reinterpret_cast<const v4i*>(sB + n * 16 * 128 + at);
#pragma unroll
            for (int m = 0; m < MT; ++m) fa[m] = *reinterpret_cast<const v4i*>(sA + m * 16 * 128 + at);
            if constexpr (decltype(last_c)::value) {
                // this group's last step is K's: products past K are zero; it may have none in this turn
                const int left = t >= steps ? 0 : t * KS + ks == KB - 1 ? rest : 128;
                if (h * 64 + 16 * g >= left) {
#pragma unroll
                    for (int m = 0; m < MT; ++m) fa[m] = (v4i){0, 0, 0, 0};
                }
            }
#pragma unroll
            for (int m = 0; m < MT; ++m)
#pragma unroll
                for (int n = 0; n < NT; ++n) acc[m][n] = mfma_i8(fb[n], fa[m], acc[m][n]);
        }
        cur = cur + 1 == STAGES ? 0 : cur + 1;
    };
    for (int t = 0; t < turns - 1; ++t) turn(t, IntC<0>{});
    turn(turns - 1, IntC<1>{});
    sum_groups<KS, MT, NT>(smem, ks, wave, acc);
    if (ks > 0) return;
    store_tiles<T>(p, row0, nrows, wm * (BM / 2), n0 + wn * (BN / 2), vec, acc, scales);
}

template <class T, int BM, int BN, int STAGES, int KS>
__global__ __launch_bounds__(256 * KS) void int8_tile_kernel(Int8Call p, int ntiles, int vec) {
    __shared__ __attribute__((aligned(1024))) uint8_t smem[KS * STAGES * (BM + BN) * 128];
    static_assert(sizeof(smem) <= 160 * 1024 && (KS - 1) * BM * BN * 4 <= (int)sizeof(smem), "LDS budget");
    Tiles x;
    const int mt = blockIdx.x / ntiles, n0 = (int)(blockIdx.x % ntiles) * BN;
    if (!find_expert<BM>(p, mt, x)) return zero_rest<T>(p, vec);
    const int64_t row0 = (int64_t)x.row + (int64_t)(mt - x.first) * BM;
    const int nrows = (int)min((int64_t)BM, x.end - row0);
    // Weights that no other row tile reads, of more than the last cache holds
    // (32 experts of 4096 x 7168, 64 rows each: 177 -> 164 us; with two row
    // tiles or more, or weights that stay cached from call to call, it costs).
    if (x.tiles == 1 && p.b_large)
        tile_run<T, BM, BN, STAGES, KS, true>(p, smem, x.e, row0, nrows, n0, vec);
    else
        tile_run<T, BM, BN, STAGES, KS, false>(p, smem, x.e, row0, nrows, n0, vec);
    zero_rest<T>(p, vec);
}

template <int BM, int BN, int STAGES, int KS>
hipError_t launch(const Int8Call& p, int out_dtype, bool vec, hipStream_t s) {
    return by_out_type(out_dtype, [&](auto t) {
        const int64_t nt = (p.N + BN - 1) / BN, tiles = max_tiles(p.rows, BM, p.E) * nt;
        hipLaunchKernelGGL((int8_tile_kernel<decltype(t), BM, BN, STAGES, KS>), dim3((unsigned)tiles), dim3(256 * KS),
                           0, s, p, (int)nt, (int)vec);
        return hipGetLastError();
    });
}

hipError_t launch_int8_tile(const Int8Call& p, int out_dtype, Int8Tile tile, bool vec, hipStream_t s) {
    switch (tile) {
        case Int8Tile::T32x32: return launch<32, 32, 4, 4>(p, out_dtype, vec, s);
        case Int8Tile::T32x64: return launch<32, 64, 3, 4>(p, out_dtype, vec, s);
        case Int8Tile::T64x64_K2: return launch<64, 64, 3, 2>(p, out_dtype, vec, s);
        case Int8Tile::T64x64: return launch<64, 64, 3, 1>(p, out_dtype, vec, s);
        case Int8Tile::T64x128_K2: return launch<64, 128, 3, 2>(p, out_dtype, vec, s);
        case Int8Tile::T64x128: return launch<64, 128, 3, 1>(p, out_dtype, vec, s);
        case Int8Tile::T128x128_K2: return launch<128, 128, 2, 2>(p, out_dtype, vec, s);
        default: return launch<128, 128, 2, 1>(p, out_dtype, vec, s);
    }
}

}  // namespace miexp
