// Products of more rows with 4-bit weights: tiles staged through LDS, with K
// shared by groups of waves where there are few tiles.
//
// A step is 128 values of K. KS groups of WM x WN waves take every KS-th step
// each. A wave multiplies 16 MT rows by 16 NT channels: it makes 16 bits of its
// weights in registers (once a step: MT row tiles share them), reads the rows'
// fragments from LDS (NT channel tiles share them), and adds each group's sums,
// scaled, to its results. Per v_mfma_f32_16x16x32 of 16 cycles that takes
// 256 / NT bytes of LDS a cycle and CU (of 128), and 52 / MT (bfloat16) and 16 /
// GS cycles of a SIMD's other instructions (GS: its products per group).
// So the smallest tiles are bound by making weights (a step of a wave with 16
// rows x 16 channels takes about 530 cycles, whatever the memory's latency: each
// SIMD's two to four waves take turns), those between by copies of rows too (about
// 20 bytes a cycle and CU), and experts' weights that are read once by memory: 64
// tokens, 8 of 256 experts each, 32 of them here, 4096 x 7168: 91 us with 16 x 128
// (425 MB of weights, 4.7 TB/s), 97 with three stages, 125 with 32 x 64.
//
// LDS rows are 256 bytes, 16-byte chunk c of row r at position c ^ (r % 16);
// weight tiles lie as in memory. Copies past K read the step's first chunk, and
// fragments past it are cut to zeros; rows past the tile repeat its last one and
// are not stored.
#include "int4_common.hpp"
#include "lds_copy.hpp"

namespace miexp {

using mimoe::g2l16s;
using mimoe::g2l4s;
using mimoe::swz16;

template <int N>
__device__ __forceinline__ void wait_copies() {
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}

template <class ST, int GS, int MT, int NT, int WM, int WN, int STAGES, int KS>
struct Int4Shape {
    static constexpr int BM = 16 * MT * WM, BN = 16 * NT * WN, WAVES = WM * WN, G = 4 / GS;
    static constexpr int X = BM * 256, W = BN * 64, S = (G * BN * (int)sizeof(ST) + 255) / 256 * 256;
    static constexpr int STAGE = X + W + S;
    static constexpr int LDS = KS * STAGES * STAGE;
    // copies of a wave and step: of 4 rows, a weight tile, and 256 bytes of scales; where there are fewer than
    // waves, some waves make the same one
    static constexpr int XC = (BM / 4 + WAVES - 1) / WAVES, WC = (BN / 16 + WAVES - 1) / WAVES,
                         SC = (S / 256 + WAVES - 1) / WAVES, LD = XC + WC + SC;
    static_assert(LDS <= 160 * 1024 && (KS - 1) * BM * BN * 4 <= LDS, "LDS budget");
};

template <class XT, class ST, int GS, int MT, int NT, int WM, int WN, int STAGES, int KS>
__global__ __launch_bounds__(64 * WM * WN * KS, WM * WN * KS <= 8 ? 2 : WM * WN * KS / 4)
void int4_tile_kernel(Int4Call p, int ntiles, int vec) {
    typedef Int4Shape<ST, GS, MT, NT, WM, WN, STAGES, KS> Z;
    typedef Operand<XT> Op;
    typedef typename Op::frag frag;
    constexpr int BM = Z::BM, BN = Z::BN, WAVES = Z::WAVES, G = Z::G, LD = Z::LD;
    __shared__ __attribute__((aligned(1024))) uint8_t smem[Z::LDS];
    if (!is_for_rows(p)) return;
    Tiles tile;
    const int mt = blockIdx.x / ntiles, n0 = (int)(blockIdx.x % ntiles) * BN;
    if (!find_expert<BM>(p, mt, tile)) return zero_rest_any(p, vec);
    const int64_t row0 = (int64_t)tile.row + (int64_t)(mt - tile.first) * BM;
    const int nrows = (int)min((int64_t)BM, tile.end - row0), e = tile.e;
    const int lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane((threadIdx.x >> 6) % WAVES);
    const int ks = __builtin_amdgcn_readfirstlane((threadIdx.x >> 6) / WAVES);
    const int wm = wave % WM, wn = wave / WM;
    const int rest = p.K - (p.KT - 1) * 128;  // values of the last step: 8 .. 128

    // Rows: copy i of a wave fills 4 LDS rows; lane l takes row l / 16, position
    // l % 16. An id that is no row reads row 0, and is not used.
    const uint8_t* x_base = (const uint8_t*)p.x + (p.row_ids ? 0 : row0 * p.x_stride * 2);
    uint32_t x_off[Z::XC], x_cut[Z::XC];
#pragma unroll
    for (int i = 0; i < Z::XC; ++i) {
        const int row = 4 * ((wave + i * WAVES) % (BM / 4)) + (lane >> 4), chunk = (lane & 15) ^ swz16(row);
        const int m = min(row, nrows - 1);
        const int64_t from = p.row_ids ? max(source_row(p, row0 + m), (int64_t)0) : m;
        x_off[i] = (uint32_t)(from * p.x_stride) * 2 + chunk * 16;
        x_cut[i] = chunk * 8 >= rest ? chunk * 16 : 0;
    }
    // Weights: a row of tiles for each copy; those past the last repeat it.
    const uint8_t* w_base = p.w + e * p.w_expert;
    const int last_tile = p.Np / 16 - 1;
    // Scales: dword d of a stage is that of channels d % D of group d / D.
    constexpr int D = BN * (int)sizeof(ST) / 4;
    const uint8_t* s_base = (const uint8_t*)p.scale + (e * p.scale_expert + n0) * (int64_t)sizeof(ST);
    const int row_bytes = p.Np * (int)sizeof(ST), last_group = (p.K - 1) >> p.group_shift;
    uint8_t* mine = smem + ks * STAGES * Z::STAGE;
    auto issue = [&](int kb, int stage) __attribute__((always_inline)) {
        uint8_t* to = mine + stage * Z::STAGE;
        const uint8_t* x = x_base + (int64_t)kb * 256;
        const uint32_t last = kb == p.KT - 1 ? ~0u : 0u;
#pragma unroll
        for (int i = 0; i < Z::XC; ++i)
            g2l16s(x, x_off[i] - (x_cut[i] & last), to + ((wave + i * WAVES) % (BM / 4)) * 1024);
#pragma unroll
        for (int i = 0; i < Z::WC; ++i) {
            const int t = (wave + i * WAVES) % (BN / 16);
            g2l16s(w_base + ((int64_t)min(n0 / 16 + t, last_tile) * p.KT + kb) * 1024, lane * 16, to + Z::X + t * 1024);
        }
#pragma unroll
        for (int i = 0; i < Z::SC; ++i) {
            const int c = (wave + i * WAVES) % (Z::S / 256), d = c * 64 + lane;
            const int row = min(G == 1 ? (kb * 128) >> p.group_shift : kb * G + d / D, last_group);
            g2l4s(s_base, (uint32_t)row * row_bytes + min(d % D * 4, row_bytes - n0 * (int)sizeof(ST) - 4),
                  to + Z::X + Z::W + c * 256);
        }
    };

    v4f acc[MT][NT];
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int n = 0; n < NT; ++n) acc[m][n] = (v4f){0.f, 0.f, 0.f, 0.f};
    // turn t: step t * KS + ks of K, in buffer t % STAGES
    const int turns = (p.KT + KS - 1) / KS, steps = p.KT > ks ? (p.KT - ks - 1) / KS + 1 : 0;  // of this group
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
        const uint8_t* sx = mine + cur * Z::STAGE + wm * MT * 4096;
        const uint8_t* sw = mine + cur * Z::STAGE + Z::X + wn * NT * 1024;
        const uint8_t* ss = mine + cur * Z::STAGE + Z::X + Z::W + wn * NT * 16 * sizeof(ST);
        typedef ST s4 __attribute__((ext_vector_type(4)));
        cur = cur + 1 == STAGES ? 0 : cur + 1;
        // this group's last step may be K's: products past K are zero; it may have none in this turn
        const int left = !decltype(last_c)::value ? 128 : t >= steps ? 0 : t * KS + ks == p.KT - 1 ? rest : 128;
        if (decltype(last_c)::value && left == 0) return;
        // The compiler would sink each LDS read to its use and wait there for it: what
        // a fence of the scheduler parts stays in this order.
        auto fence = [] { __builtin_amdgcn_sched_barrier(0); };
        frag w[NT][4], x[2][4];
        v4f scale[NT][G];
        v4u d[NT];
        s4 s[NT][G];
        auto fragments = [&](int m) __attribute__((always_inline)) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                x[m & 1][i] = *reinterpret_cast<const frag*>(sx + (m * 16 + r) * 256 + ((4 * i + g) ^ r) * 16);
                if (decltype(last_c)::value && 32 * i + 8 * g >= left) x[m & 1][i] = __builtin_bit_cast(frag, (v4u){0, 0, 0, 0});
            }
        };
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            d[n] = *reinterpret_cast<const v4u*>(sw + n * 1024 + lane * 16);
#pragma unroll
            for (int j = 0; j < G; ++j) s[n][j] = *reinterpret_cast<const s4*>(ss + (j * BN + n * 16 + 4 * g) * sizeof(ST));
        }
        fragments(0);
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
#pragma unroll
        for (int m = 0; m < MT; ++m) {
            fence();
            if (m + 1 < MT) fragments(m + 1);
            fence();
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
    };
    for (int t = 0; t < turns - 1; ++t) turn(t, IntC<0>{});
    turn(turns - 1, IntC<1>{});
    // Sums of the groups that shared K, in group 0.
    if constexpr (KS > 1) {
        v4f* red = reinterpret_cast<v4f*>(smem);
        __syncthreads();
        if (ks > 0) {
#pragma unroll
            for (int m = 0; m < MT; ++m)
#pragma unroll
                for (int n = 0; n < NT; ++n) red[(((ks - 1) * WAVES + wave) * MT * NT + m * NT + n) * 64 + lane] = acc[m][n];
        }
        __syncthreads();
        if (ks == 0) {
            for (int k = 0; k < KS - 1; ++k)
#pragma unroll
                for (int m = 0; m < MT; ++m)
#pragma unroll
                    for (int n = 0; n < NT; ++n) acc[m][n] += red[((k * WAVES + wave) * MT * NT + m * NT + n) * 64 + lane];
        }
    }
    if (ks == 0) {
#pragma unroll
        for (int m = 0; m < MT; ++m) {
            const int row = (wm * MT + m) * 16 + r;
            if (row >= nrows) continue;
#pragma unroll
            for (int n = 0; n < NT; ++n) store_sums<Op>(p, row0 + row, n0 + (wn * NT + n) * 16 + 4 * g, vec, acc[m][n]);
        }
    }
    zero_rest_any(p, vec);
}

template <int MT, int NT, int WM, int WN, int STAGES, int KS>
hipError_t launch(const Int4Call& p, int x_dtype, int scale_dtype, bool vec, hipStream_t s) {
    return by_int4_types(x_dtype, scale_dtype, 1 << p.group_shift, [&](auto x, auto sc, auto gs) {
        constexpr int GS = decltype(gs)::value;
        constexpr int BM = 16 * MT * WM, BN = 16 * NT * WN;
        // a launch that is for at most so many rows needs no more workgroups
        const int64_t nt = (p.N + BN - 1) / BN, rows = p.rows < p.to_rows ? p.rows : p.to_rows;
        const int64_t tiles = max_tiles(rows, BM, p.E) * nt;
        hipLaunchKernelGGL((int4_tile_kernel<decltype(x), decltype(sc), GS, MT, NT, WM, WN, STAGES, KS>),
                           dim3((unsigned)tiles), dim3(64 * WM * WN * KS), 0, s, p, (int)nt, (int)vec);
        return hipGetLastError();
    });
}

hipError_t launch_int4_tile(const Int4Call& p, int x_dtype, int scale_dtype, Int4Tile tile, bool vec, hipStream_t s) {
    switch (tile) {
        case Int4Tile::T16x32: return launch<1, 1, 1, 2, 5, 4>(p, x_dtype, scale_dtype, vec, s);
        case Int4Tile::T16x64: return launch<1, 1, 1, 4, 4, 2>(p, x_dtype, scale_dtype, vec, s);
        case Int4Tile::T16x128: return launch<1, 2, 1, 4, 2, 2>(p, x_dtype, scale_dtype, vec, s);
        case Int4Tile::T32x64: return launch<2, 1, 1, 4, 3, 2>(p, x_dtype, scale_dtype, vec, s);
        case Int4Tile::T32x128: return launch<2, 2, 1, 4, 2, 2>(p, x_dtype, scale_dtype, vec, s);
        case Int4Tile::T64x64: return launch<4, 1, 1, 4, 3, 2>(p, x_dtype, scale_dtype, vec, s);
        case Int4Tile::T64x128: return launch<4, 2, 1, 4, 3, 2>(p, x_dtype, scale_dtype, vec, s);
        default: return launch<4, 2, 2, 4, 3, 1>(p, x_dtype, scale_dtype, vec, s);
    }
}

}  // namespace miexp
