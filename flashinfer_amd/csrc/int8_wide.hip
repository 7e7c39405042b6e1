// Integer products of many rows, in tiles of 256 rows x 256 channels: one
// workgroup per CU, its eight waves in two groups that take turns at the
// matrix cores.
//
// Waves 0-3 (group 0) and 4-7 (group 1) share the four SIMDs, one wave of each
// group per SIMD; wave wn of a group owns 64 channels. Rows go in blocks of
// 64: group G has blocks G and 2 + G. A step of 128 bytes of K is four phases
// per wave, a barrier after each, and group 1 runs one phase behind group 0:
//   M0: read the weight fragments and block G's rows from LDS
//   C0: their 32 MFMAs
//   M1: read block 2 + G's rows
//   C1: their 32 MFMAs
// so one wave of a SIMD multiplies from registers while the other one reads
// LDS and issues copies. A tile of at most 128 rows has M0 and C0 alone.
//
// Copies (two stages): B0 = the weights and rows 0-127 of a step, B1 = rows
// 128-255. B0 of step kb + 2 goes out in M1 of kb, after both groups have read
// that of kb; B1 of kb + 1 in M0 of kb. What the next slot's readers need is
// waited for by the wave that issued it (the NV copies issued since may stay
// in flight) before the barrier that ends the slot: for group 0 that is the
// end of C0 / C1, for group 1, one slot behind, the end of M0 / M1. Past a
// tile's last step the copies go on with the next tile's first ones (its B0,
// B1 of step 0, B0 of step 1), so a tile starts with its operands there, and
// one group stores its results while the other still multiplies.
//
// Results go through LDS, a wave's 16 rows at a time, so that stores cover
// whole 128-byte lines (8192 x 8192 x 1024: 86 us, 121 with a store per MFMA
// tile and a workgroup per tile).
//
// 8192 x 4096 x 7168 185-189 us (2.6 POP/s; a loop of nothing but these MFMAs
// on random data reaches 3.2, held by power), 4096 x 4096 x 7168 91 us. A step
// takes about 3,300 cycles, 2,048 of them MFMA. No one part holds it: where the
// whole takes 204 us, it is 178 without the copies, 188 without the LDS reads
// and 140 without the MFMAs, so what is left is in the slots' ends. Experts'
// products with few rows each are bound as much by their weights: 8192 rows
// over 32 experts of 7168 x 2048, drawn evenly, 190-194 us for 604 MB and 0.24
// TOP (159 with exactly 256 rows each, a tile of rows); on a box where it took
// 207-224, 173 without the copies and 177 without the MFMAs.
//
// Measured and left out: four waves of 128 x 128 (a third fewer LDS reads, but
// copies only half a step ahead: 245 us), phases by halves of K instead of rows
// (evenly long, copies a step ahead: 230), reading the second halves during the
// C phases (214), 32 x 32 x 32 MFMAs (5 % faster by themselves; 228 against
// 204), weights from memory into registers (neighbouring lanes read different
// rows: 313 against 203), shares of tiles by cost or from a queue (no faster:
// tiles of few rows cost as much as full ones, their weights).
#include "int8_common.hpp"

namespace miexp {

using mimoe::g2l16;
using mimoe::g2l16s;
using mimoe::g2l4;
using mimoe::swzq;

namespace wide {
constexpr int BM = 256, BN = 256, GM = 8;
constexpr int A_BYTES = 128 * 128, B_BYTES = BN * 128, STAGE = 2 * A_BYTES + B_BYTES;
constexpr int NV = 4 + 2 + 2;         // copies of a wave and step: weights, rows, rows
constexpr int OUT_LD = 128 + 16;      // bytes of a row of results in LDS
constexpr int OUT_BYTES = 16 * OUT_LD;  // of a wave
struct Lds {
    uint8_t stage[2][STAGE];
    uint8_t out[8][OUT_BYTES];
    float scale[2][BM + 2 * BN];  // of the tile's rows and channels, and biases; two tiles overlap
};
static_assert(sizeof(Lds) <= 160 * 1024, "LDS budget");
}  // namespace wide

// End of a phase: this wave's LDS reads are done and at most N of its copies
// are in flight; then the workgroup's barrier.
template <int N>
__device__ __forceinline__ void phase_end() {
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(N) : "memory");
}
__device__ __forceinline__ void phase_end() {
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
}

struct WideTile {
    int e, n0, nrows;
    int64_t row0;
};

// The whole run of one wave of group G over its workgroup's tiles
// first, first + step, .. below end.
template <class T, int G>
__device__ __forceinline__ void wide_run(const Int8Call& p, wide::Lds& lds, int ntiles, int first, int end, int step,
                                         bool vec16) {
    using namespace wide;
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wn = wave & 3;
    const int r = lane & 15, g = lane >> 4;
    const int KB = (p.K + 127) / 128;

    auto tile = [&](int t) __attribute__((always_inline)) {
        WideTile w;
        int nt;
        tile_at<BM, GM>(p, t, ntiles, w.e, w.row0, w.nrows, nt);
        w.n0 = nt * BN;
        return w;
    };
    // A copy fills 8 LDS rows: lane l takes row l / 8, position l % 8, which
    // holds chunk (l % 8) ^ swzq(row). Its source is a base in SGPRs (the
    // tile's first row; a itself with row_ids) and a 32-bit offset of the lane.
    // Past K, in a last step that K ends in, lanes read zeros. An id that is
    // no row reads row 0: its scale is NaN.
    auto chunk = [&](int l, int row) __attribute__((always_inline)) { return ((l & 7) ^ swzq(row)) * 16; };
    auto a_row = [&](int l, int i) __attribute__((always_inline)) {  // of copy i: 0, 1 rows 0-127; 2, 3 rows 128-255
        return (i >> 1) * 128 + (wave * 2 + (i & 1)) * 8 + (l >> 3);
    };
    auto b_row = [&](int l, int i) __attribute__((always_inline)) { return 8 * (wave * 4 + i) + (l >> 3); };
    // The lane number, as a value of its own wherever it is asked for: what is
    // made of it is then computed there and takes no register in between.
    auto here = [&]() __attribute__((always_inline)) {
        int l = lane;
        asm volatile("" : "+v"(l));
        return l;
    };
    const int rest = p.K - (KB - 1) * 128;  // bytes of the last step: 16 .. 128
    const int8_t *a_base[2], *b_base;
    uint32_t a_off[4], b_off[4], a_next[4];  // a_next: those of the next tile
    auto find_rows = [&](const WideTile& w) __attribute__((always_inline)) {
        const int l = here();
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int row = min(a_row(l, i), w.nrows - 1);
            const int64_t from = p.row_ids ? max(source_row(p, w.row0 + row), (int64_t)0) : row;
            a_next[i] = (uint32_t)(from * p.a_stride) + chunk(l, a_row(l, i));
        }
    };
    auto point_a = [&](const WideTile& w, int half) __attribute__((always_inline)) {
        a_base[half] = p.a + (p.row_ids ? 0 : w.row0 * p.a_stride);
#pragma unroll
        for (int i = 2 * half; i < 2 * half + 2; ++i) a_off[i] = a_next[i];
    };
    auto point_b = [&](const WideTile& w) __attribute__((always_inline)) {
        b_base = p.b + w.e * p.b_expert_stride + (int64_t)w.n0 * p.b_stride;
        const int l = here();
#pragma unroll
        for (int i = 0; i < 4; ++i)
            b_off[i] = (uint32_t)(min(b_row(l, i), p.N - 1 - w.n0) * p.b_stride) + chunk(l, b_row(l, i));
    };
    auto issue_b0 = [&](int kb, int s) __attribute__((always_inline)) {
        uint8_t* dst = lds.stage[s] + wave * 2048;
        uint8_t* dst_b = lds.stage[s] + 2 * A_BYTES + wave * 4096;
        const int8_t *a = a_base[0] + kb * 128, *b = b_base + kb * 128;
        if (kb < KB - 1 || rest == 128) {
#pragma unroll
            for (int i = 0; i < 4; ++i) g2l16s(b, b_off[i], dst_b + i * 1024);
#pragma unroll
            for (int i = 0; i < 2; ++i) g2l16s(a, a_off[i], dst + i * 1024);
        } else {
            const int l = here();
#pragma unroll
            for (int i = 0; i < 4; ++i)
                g2l16(chunk(l, b_row(l, i)) < rest ? (const void*)(b + b_off[i]) : (const void*)&kZeros, dst_b + i * 1024);
#pragma unroll
            for (int i = 0; i < 2; ++i)
                g2l16(chunk(l, a_row(l, i)) < rest ? (const void*)(a + a_off[i]) : (const void*)&kZeros, dst + i * 1024);
        }
    };
    auto issue_b1 = [&](int kb, int s) __attribute__((always_inline)) {
        uint8_t* dst = lds.stage[s] + A_BYTES + wave * 2048;
        const int8_t* a = a_base[1] + kb * 128;
        if (kb < KB - 1 || rest == 128) {
#pragma unroll
            for (int i = 0; i < 2; ++i) g2l16s(a, a_off[2 + i], dst + i * 1024);
        } else {
            const int l = here();
#pragma unroll
            for (int i = 0; i < 2; ++i)
                g2l16(chunk(l, a_row(l, 2 + i)) < rest ? (const void*)(a + a_off[2 + i]) : (const void*)&kZeros,
                      dst + i * 1024);
        }
    };

    // fragment of 16 rows at s: this lane's row r, 16-byte chunks g and g + 4
    const int lo_off = r * 128 + ((g ^ swzq(r)) << 4), hi_off = r * 128 + (((g + 4) ^ swzq(r)) << 4);
    v4i bfr[4][2], afr[4][2];
    auto frag = [&](v4i (&f)[2], const uint8_t* s) __attribute__((always_inline)) {
        f[0] = *reinterpret_cast<const v4i*>(s + lo_off);
        f[1] = *reinterpret_cast<const v4i*>(s + hi_off);
    };
    auto read_b0 = [&](int s) __attribute__((always_inline)) {
        const uint8_t* st = lds.stage[s];
#pragma unroll
        for (int n = 0; n < 4; ++n) frag(bfr[n], st + 2 * A_BYTES + (wn * 64 + n * 16) * 128);
#pragma unroll
        for (int m = 0; m < 4; ++m) frag(afr[m], st + (G * 64 + m * 16) * 128);
        __builtin_amdgcn_sched_barrier(0);
    };
    auto read_b1 = [&](int s) __attribute__((always_inline)) {
#pragma unroll
        for (int m = 0; m < 4; ++m) frag(afr[m], lds.stage[s] + A_BYTES + (G * 64 + m * 16) * 128);
        __builtin_amdgcn_sched_barrier(0);
    };
    v4i acc[8][4];
    // C phase. The empty asm statements keep the compiler from sinking MFMAs
    // below the barrier.
    auto multiply = [&](v4i (*c)[4]) __attribute__((always_inline)) {
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int m = 0; m < 4; ++m)
#pragma unroll
                for (int n = 0; n < 4; ++n) c[m][n] = mfma_i8(bfr[n][h], afr[m][h], c[m][n]);
#pragma unroll
        for (int m = 0; m < 4; ++m)
            asm volatile("" : "+v"(c[m][0]), "+v"(c[m][1]), "+v"(c[m][2]), "+v"(c[m][3]));
        __builtin_amdgcn_sched_barrier(0);
    };
    // Results of 64 rows: block `b` of the tile, 128 bytes of each row at a time.
    auto store_block = [&](const WideTile& w, int b, const float* scale, const v4i (*c)[4])
        __attribute__((always_inline)) {
        if (b * 64 >= w.nrows) return;
        constexpr int NP = 8 / sizeof(T);  // channel tiles of 128 bytes of a row
        constexpr int PER = 16 / sizeof(T);
        uint8_t* buf = lds.out[wave];
        const int l = here(), r = l & 15, g = l >> 4;
        const int row = l >> 3, col = (l & 7) * PER;  // what this lane stores: rows row and 8 + row
#pragma unroll
        for (int n0 = 0; n0 < 4; n0 += NP) {
            float sb[NP][4], bias[NP][4];
#pragma unroll
            for (int n = 0; n < NP; ++n)
#pragma unroll
                for (int v = 0; v < 4; ++v) {
                    sb[n][v] = scale[BM + wn * 64 + (n0 + n) * 16 + 4 * g + v];
                    bias[n][v] = scale[BM + BN + wn * 64 + (n0 + n) * 16 + 4 * g + v];
                }
            const int n_at = w.n0 + wn * 64 + n0 * 16 + col;
            T* out = reinterpret_cast<T*>(p.out) + (w.row0 + b * 64 + row) * p.out_stride + n_at;
#pragma unroll
            for (int m = 0; m < 4; ++m) {
                const float sa = scale[b * 64 + m * 16 + r];
#pragma unroll
                for (int n = 0; n < NP; ++n) {
                    float y[4];
#pragma unroll
                    for (int v = 0; v < 4; ++v) y[v] = (float)c[m][n0 + n][v] * sa * sb[n][v] + bias[n][v];
                    store<T, 4>(reinterpret_cast<T*>(buf + r * OUT_LD) + n * 16 + 4 * g, y);
                }
                __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
                __builtin_amdgcn_wave_barrier();
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const v4i v = *reinterpret_cast<const v4i*>(buf + (h * 8 + row) * OUT_LD + col * sizeof(T));
                    if (b * 64 + m * 16 + h * 8 + row >= w.nrows) continue;
                    T* to = out + (m * 16 + h * 8) * p.out_stride;
                    if (vec16) {
                        if (n_at < p.N) *reinterpret_cast<v4i*>(to) = v;
                    } else {
                        const typename Vec<T, PER>::type x = __builtin_bit_cast(typename Vec<T, PER>::type, v);
#pragma unroll
                        for (int i = 0; i < PER; ++i)
                            if (n_at + i < p.N) to[i] = x[i];
                    }
                }
                __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
                __builtin_amdgcn_wave_barrier();
            }
        }
    };

    int t = first;
    WideTile w = tile(t);
    find_rows(w);
    point_a(w, 0);
    point_a(w, 1);
    point_b(w);
    issue_b0(0, 0);
    issue_b1(0, 0);
    issue_b0(1, 1);
    phase_end<NV>();
    if constexpr (G == 1) phase_end();
    int s = 0, turn = 0;  // stage of the tile's first step; which scales
    for (;;) {
        // here: B0(0), B1(0), B0(1) have gone out, and B0(0) has landed
        const bool more = t + step < end;
        WideTile next = w;
        if (more) next = tile(t + step);
        find_rows(next);
        // Scales: channels (and biases) by group 0, rows by group 1. They are
        // waited for with the copies.
        float* scale = lds.scale[turn];
        if constexpr (G == 0) {
            const int l = here(), n = min(w.n0 + wn * 64 + l, p.N - 1);
            g2l4(p.b_scale + (int64_t)w.e * p.N + n, scale + BM + wn * 64);
            scale[BM + BN + wn * 64 + l] = bias_at(p, n);
        } else {
            const int64_t id = source_row(p, w.row0 + min(wn * 64 + here(), w.nrows - 1));
            g2l4(id >= 0 ? p.a_scale + id : &kNan, scale + wn * 64);
        }
#pragma unroll
        for (int m = 0; m < 8; ++m)
#pragma unroll
            for (int n = 0; n < 4; ++n) acc[m][n] = (v4i){0, 0, 0, 0};
        const bool large = w.nrows > 128, second = (2 + G) * 64 < w.nrows;
        // Small tiles: B0 of step kb goes out in the slot after both groups
        // have read step kb - 2: M0 of kb - 1 for group 0, C0 of kb - 2 for group 1.
        auto past = [&](int kb) __attribute__((always_inline)) {
            if (kb == KB) {
                point_a(next, 0);
                point_b(next);
            }
            if (kb == KB + 1) {
                point_a(next, 1);
                issue_b1(0, G == 0 ? s : s ^ 1);  // stage of step KB
            }
            issue_b0(kb >= KB ? kb - KB : kb, G == 0 ? s ^ 1 : s);
        };
#pragma unroll 1
        for (int kb = 0; kb < KB; ++kb, s ^= 1) {
            // M0
            read_b0(s);
            if (large) {
                if (kb == KB - 1) point_a(next, 1);
                issue_b1(kb == KB - 1 ? 0 : kb + 1, s ^ 1);
                __builtin_amdgcn_sched_barrier(0);
                if constexpr (G == 1) phase_end<NV>(); else phase_end();
            } else {
                if constexpr (G == 0) {
                    if (kb > 0) past(kb + 1);
                }
                __builtin_amdgcn_sched_barrier(0);
                if constexpr (G == 1) {
                    phase_end<0>();
                    past(kb + 2);
                } else {
                    phase_end();
                }
            }
            // C0
            multiply(acc);
            if (!large) {
                if constexpr (G == 0) phase_end<0>(); else phase_end();
                continue;
            }
            if constexpr (G == 0) phase_end<NV>(); else phase_end();
            // M1
            read_b1(s);
            if (kb == KB - 2) {
                point_a(next, 0);
                point_b(next);
            }
            issue_b0(kb + 2 >= KB ? kb + 2 - KB : kb + 2, s);
            __builtin_amdgcn_sched_barrier(0);
            if constexpr (G == 1) phase_end<NV>(); else phase_end();
            // C1
            if (second) multiply(acc + 4);
            if constexpr (G == 0) phase_end<NV>(); else phase_end();
        }
        if constexpr (G == 0) {
            if (!large) past(KB + 1);
        }
        if constexpr (G == 0) {
            if (!more) phase_end();  // group 1's last phase
        }
        store_block(w, G, scale, acc);
        store_block(w, 2 + G, scale, acc + 4);
        if (!more) break;
        t += step;
        w = next;
        turn ^= 1;
    }
    mimoe::wait_vmem();  // no copy into LDS may be pending when the workgroup ends
}

template <class T>
__global__ __launch_bounds__(512) void int8_wide_kernel(Int8Call p, int ntiles, int vec16) {
    __shared__ __attribute__((aligned(1024))) wide::Lds lds;
    const int total = count_tiles<wide::BM>(p) * ntiles;
    // each of the 8 XCDs (workgroup b runs on b % 8) takes one contiguous eighth of the order
    const int per_xcd = (total + 7) >> 3, xcd = blockIdx.x & 7;
    const int first = xcd * per_xcd + (blockIdx.x >> 3), end = min(total, (xcd + 1) * per_xcd);
    if (first < end) {
        if (threadIdx.x < 256)
            wide_run<T, 0>(p, lds, ntiles, first, end, gridDim.x >> 3, vec16);
        else
            wide_run<T, 1>(p, lds, ntiles, first, end, gridDim.x >> 3, vec16);
    }
    zero_rest<T>(p, vec16);
}

// K > 128: two steps at least.
hipError_t launch_int8_wide(const Int8Call& p, int out_dtype, hipStream_t s) {
    return by_out_type(out_dtype, [&](auto t) {
        typedef decltype(t) T;
        const int64_t nt = (p.N + wide::BN - 1) / wide::BN, tiles = (max_tiles(p.rows, wide::BM, p.E) * nt + 7) / 8 * 8;
        const int per16 = 16 / (int)sizeof(T);
        const bool vec16 = (uint64_t)p.out % 16 == 0 && p.out_stride % per16 == 0 && p.N % per16 == 0;
        hipLaunchKernelGGL(int8_wide_kernel<T>, dim3((unsigned)(tiles < 256 ? tiles : 256)), dim3(512), 0, s, p,
                           (int)nt, (int)vec16);
        return hipGetLastError();
    });
}

}  // namespace miexp
