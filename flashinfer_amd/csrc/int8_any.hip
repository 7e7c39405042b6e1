// Integer products whose rows lie at any address: K, strides and pointers that
// are no multiples of 16.
//
// The tiles of int8_tile.hip, but with operands that go through registers:
// 16 bytes of a row at a time, loaded from whatever address they have (the
// hardware splits those that cross a line), written to LDS as aligned rows one
// turn later. A row's last 1 to 15 bytes are the end of the 16 bytes before
// its end, shifted down; a row of fewer than 16 is put together byte by byte.
// Costs against aligned rows: 16 x 4096 x 7169 15.2 us (K = 7168 8.5), 1000 x
// 1000 x 1000 7.3 (K = 1008 6.6), 8192 x 4096 x 7169 414 (189), which is why
// large dense products with such a K are copied first (int8_gemm.hip). Others
// of any size come here as they are: those whose strides or addresses alone are
// off (8192 x 4096 x 7168 with one operand a byte off: 332), grouped ones, and
// gathers from 2^32 bytes and more.
#include "int8_common.hpp"

namespace miexp {

using mimoe::swzq;

typedef v4i v4i_u __attribute__((aligned(1)));

// Bytes k .. k + 15 of the row of K bytes at p; zeros past its end.
__device__ __forceinline__ v4i row16(const int8_t* p, int k, int K) {
    const int left = K - k;
    if (left >= 16) return *reinterpret_cast<const v4i_u*>(p + k);
    if (left <= 0) return (v4i){0, 0, 0, 0};
    unsigned __int128 x = 0;
    if (K >= 16) {
        x = __builtin_bit_cast(unsigned __int128, (v4i)*reinterpret_cast<const v4i_u*>(p + K - 16));
        x >>= 8 * (16 - left);
    } else {
        for (int i = 0; i < left; ++i) x |= (unsigned __int128)(uint8_t)p[k + i] << (8 * i);
    }
    return __builtin_bit_cast(v4i, x);
}

// Rows of K bytes at any address -> rows of ld bytes (a multiple of 16), zeros
// past K: the rows of a, then those of b.
__global__ __launch_bounds__(256) void pack_rows_kernel(Int8Call p, int8_t* __restrict__ to, int ld) {
    for (int64_t row = blockIdx.x; row < p.a_rows + p.N; row += gridDim.x) {
        const int8_t* from = row < p.a_rows ? p.a + row * p.a_stride : p.b + (row - p.a_rows) * p.b_stride;
        for (int k = threadIdx.x * 16; k < ld; k += 256 * 16)
            *reinterpret_cast<v4i*>(to + row * ld + k) = row16(from, k, p.K);
    }
}

hipError_t launch_pack_rows(const Int8Call& p, int8_t* to, int ld, hipStream_t s) {
    const int64_t rows = p.a_rows + p.N;
    hipLaunchKernelGGL(pack_rows_kernel, dim3((unsigned)(rows < MAX_BLOCKS ? rows : MAX_BLOCKS)), dim3(256), 0, s, p,
                       to, ld);
    return hipGetLastError();
}

template <class T, int BM, int BN, int KS>
__global__ __launch_bounds__(256 * KS) void int8_any_kernel(Int8Call p, int ntiles, int vec) {
    constexpr int MT = BM / 32, NT = BN / 32;        // 16 x 16 tiles of a wave
    constexpr int A_LD = BM / 32, LD = (BM + BN) / 32;  // 16-byte loads of a thread and step
    constexpr int STAGE = (BM + BN) * 128;
    __shared__ __attribute__((aligned(1024))) uint8_t smem[KS * 2 * STAGE];
    static_assert((KS - 1) * BM * BN * 4 <= (int)sizeof(smem), "LDS budget");
    int e, nrows;
    int64_t row0;
    if (!find_tile<BM>(p, blockIdx.x / ntiles, e, row0, nrows)) return zero_rest<T>(p, vec);
    const int n0 = (int)(blockIdx.x % ntiles) * BN;
    const int lane = threadIdx.x & 63, tid = threadIdx.x & 255;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int ks = __builtin_amdgcn_readfirstlane(threadIdx.x >> 8);
    const int r = lane & 15, g = lane >> 4;
    const int wm = wave & 1, wn = wave >> 1;
    const int KB = (p.K + 127) / 128;

    // Load i of a thread: LDS row 32 i + tid / 8 (rows of a first), chunk tid % 8.
    const int8_t* src[LD];
#pragma unroll
    for (int i = 0; i < LD; ++i) {
        const int row = 32 * i + (tid >> 3);
        if (i < A_LD)  // an id that is no row reads row 0: its scale is NaN
            src[i] = p.a + max(source_row(p, row0 + min(row, nrows - 1)), (int64_t)0) * p.a_stride;
        else
            src[i] = p.b + e * p.b_expert_stride + (int64_t)min(n0 + row - BM, p.N - 1) * p.b_stride;
    }
    const int chunk = tid & 7;
    v4i held[LD];
    auto fetch = [&](int kb) __attribute__((always_inline)) {
        const int k = kb * 128 + chunk * 16;
        if (kb < KB - 1) {
#pragma unroll
            for (int i = 0; i < LD; ++i) held[i] = *reinterpret_cast<const v4i_u*>(src[i] + k);
        } else if (kb == KB - 1) {
#pragma unroll
            for (int i = 0; i < LD; ++i) held[i] = row16(src[i], k, p.K);
        } else {  // no step of this group
#pragma unroll
            for (int i = 0; i < LD; ++i) held[i] = (v4i){0, 0, 0, 0};
        }
    };
    uint8_t* mine = smem + ks * 2 * STAGE;
    auto put = [&](int stage) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < LD; ++i) {
            const int row = 32 * i + (tid >> 3);
            *reinterpret_cast<v4i*>(mine + stage * STAGE + row * 128 + ((chunk ^ swzq(row)) << 4)) = held[i];
        }
    };
    Scales<MT, NT> scales;
    scales.load(p, e, row0, nrows, wm * (BM / 2), n0 + wn * (BN / 2));
    v4i acc[MT][NT];
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int n = 0; n < NT; ++n) acc[m][n] = (v4i){0, 0, 0, 0};
    // turn t: step t * KS + ks of K, in buffer t % 2
    const int turns = (KB + KS - 1) / KS;
    fetch(ks);
    put(0);
    fetch(KS + ks);
    for (int t = 0; t < turns; ++t) {
        __syncthreads();
        const uint8_t* sA = mine + (t & 1) * STAGE + wm * (BM / 2) * 128;
        const uint8_t* sB = mine + (t & 1) * STAGE + BM * 128 + wn * (BN / 2) * 128;
        if (t + 1 < turns) {
            put((t + 1) & 1);  // read last in turn t - 1
            if (t + 2 < turns) fetch((t + 2) * KS + ks);
        }
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int at = r * 128 + (((h * 4 + g) ^ swzq(r)) << 4);
            v4i fa[MT], fb[NT];
#pragma unroll
            for (int n = 0; n < NT; ++n) fb[n] = *reinterpret_cast<const v4i*>(sB + n * 16 * 128 + at);
#pragma unroll
            for (int m = 0; m < MT; ++m) fa[m] = *reinterpret_cast<const v4i*>(sA + m * 16 * 128 + at);
#pragma unroll
            for (int m = 0; m < MT; ++m)
#pragma unroll
                for (int n = 0; n < NT; ++n) acc[m][n] = mfma_i8(fb[n], fa[m], acc[m][n]);
        }
    }
    sum_groups<KS, MT, NT>(smem, ks, wave, acc);
    if (ks == 0) store_tiles<T>(p, row0, nrows, wm * (BM / 2), n0 + wn * (BN / 2), vec, acc, scales);
    zero_rest<T>(p, vec);
}

template <int BM, int BN, int KS>
hipError_t launch(const Int8Call& p, int out_dtype, bool vec, hipStream_t s) {
    return by_out_type(out_dtype, [&](auto t) {
        const int64_t nt = (p.N + BN - 1) / BN, tiles = max_tiles(p.rows, BM, p.E) * nt;
        hipLaunchKernelGGL((int8_any_kernel<decltype(t), BM, BN, KS>), dim3((unsigned)tiles), dim3(256 * KS), 0, s, p,
                           (int)nt, (int)vec);
        return hipGetLastError();
    });
}

hipError_t launch_int8_any(const Int8Call& p, int out_dtype, Int8Tile tile, bool vec, hipStream_t s) {
    switch (tile) {
        case Int8Tile::T32x32: return launch<32, 32, 4>(p, out_dtype, vec, s);
        case Int8Tile::T32x64: return launch<32, 64, 4>(p, out_dtype, vec, s);
        case Int8Tile::T64x64_K2: return launch<64, 64, 2>(p, out_dtype, vec, s);
        case Int8Tile::T64x64: return launch<64, 64, 1>(p, out_dtype, vec, s);
        case Int8Tile::T64x128_K2: return launch<64, 128, 2>(p, out_dtype, vec, s);
        case Int8Tile::T64x128: return launch<64, 128, 1>(p, out_dtype, vec, s);
        case Int8Tile::T128x128_K2: return launch<128, 128, 2>(p, out_dtype, vec, s);
        default: return launch<128, 128, 1>(p, out_dtype, vec, s);
    }
}

}  // namespace miexp
