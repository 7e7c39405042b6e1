// Slots sorted by local expert: a stable counting sort of T * k ids into E + 1
// buckets, the last of which takes the ids of other shards.
//
//   row(slot) = #{slots in lower buckets} + #{earlier slots in its bucket}
//
// The second term is found a wave at a time: lanes with equal buckets find
// each other by one ballot per bit of the bucket, a lane's place among them is
// the count of equal lanes below it, and the lowest of them advances the
// bucket's counter in LDS. Counters belong to one wave each and waves take
// contiguous slots, so the order is that of the slots and no result hangs on
// the order of atomics.
//
// Up to SMALL slots one workgroup does it all. Beyond, one launch counts the
// buckets of at most 256 chunks, and a second one places them: each workgroup
// sums the counts of the chunks before its own, which are in L2. What bounds
// it is the latency of a few dependent passes, not its 12 bytes a slot: 8
// slots 4.2 us, 2048 6.6, 4096 8.5 (9.1 in one workgroup), 8000 8.4 (21),
// 65536 13.5, a million 47 (on another box 8000 9.8, 65536 14.0, a million 48).
#include "experts_common.hpp"

namespace miexp {

constexpr int64_t SMALL = 3000;
constexpr int64_t MAX_CHUNKS = 256;

// Slots of a chunk. Short chunks shorten a wave's walk, many chunks the sums
// over them: up to 10240 slots 6 to 20 chunks of 512 (8000 slots: 8.4 us in 16,
// 9.5 in four), up to 32768 11 to 32 of 1024 (16384: 9.6 in 16, 10.7 in 32), up
// to 131072 17 to 64 of 2048 (65536: 13.5 in 32, 18.4 in 16), up to 262144 33 to
// 64 of 4096, then of 8192 and more, at most 256 (524288: 38 in 64, 43 in 256,
// 60 in 32). Where the length doubles the time hardly steps: 32768 and 32776
// slots 12.1 and 12.3 us, 131072 and 131080 18.0 and 20.4.
inline int64_t chunk_len(int64_t slots) {
    int64_t len = 512;
    while (len * (len < 1024 ? 20 : len < 2048 ? 32 : len < 8192 ? 64 : MAX_CHUNKS) < slots) len *= 2;
    return len;
}

int64_t sort_chunks(int64_t slots) {
    if (slots <= SMALL) return 0;
    const int64_t len = chunk_len(slots);
    return (slots + len - 1) / len;
}

__device__ __forceinline__ int bucket_of(int id, long long offset, int E) {
    const long long l = (long long)id - offset;
    return l >= 0 && l < E ? (int)l : E;
}

// Lanes of the wave whose bucket is this lane's, among those with `live`.
__device__ __forceinline__ unsigned long long same_bucket(int b, int bits, bool live) {
    unsigned long long m = __ballot(live);
    for (int i = 0; i < bits; ++i) {
        const unsigned long long on = __ballot((b >> i) & 1);
        m &= (b >> i) & 1 ? on : ~on;
    }
    return m;
}

// Exclusive scan over the workgroup's threads of one value each; *total gets
// the sum. `tmp` holds a value per wave.
__device__ __forceinline__ int block_scan(int v, int* tmp, int* total) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, waves = blockDim.x >> 6;
    int inc = v;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const int u = __shfl_up(inc, d);
        if (lane >= d) inc += u;
    }
    if (lane == 63) tmp[wave] = inc;
    __syncthreads();
    int before = 0, all = 0;
    for (int w = 0; w < waves; ++w) {
        const int u = tmp[w];
        if (w < wave) before += u;
        all += u;
    }
    *total = all;
    __syncthreads();
    return before + inc - v;
}

// A wave's part of the slots being placed: BATCHES of 64, kept in registers.
constexpr int BATCHES = 4;
struct Batch {
    int bucket;
    unsigned long long same;  // lanes with this lane's bucket
};

// Counts the buckets of this wave's slots [a, z) into mine[]; the first
// BATCHES of them stay in `kept`.
__device__ __forceinline__ void count_slots(const int32_t* ids, int64_t a, int64_t z, int E, long long offset,
                                            int bits, int* mine, Batch (&kept)[BATCHES]) {
    const int lane = threadIdx.x & 63;
    auto add = [&](int64_t s, int id) {
        Batch x;
        const bool live = s + lane < z;
        x.bucket = live ? bucket_of(id, offset, E) : 0;
        x.same = same_bucket(x.bucket, bits, live);
        if (live && lane == __ffsll(x.same) - 1) atomicAdd(&mine[x.bucket], __popcll(x.same));
        return x;
    };
    int id[BATCHES];
#pragma unroll
    for (int i = 0; i < BATCHES; ++i) id[i] = a + i * 64 + lane < z ? ids[a + i * 64 + lane] : 0;
#pragma unroll
    for (int i = 0; i < BATCHES; ++i)
        if (a + i * 64 < z) kept[i] = add(a + i * 64, id[i]);
    for (int64_t s = a + BATCHES * 64; s < z; s += 64) add(s, s + lane < z ? ids[s + lane] : 0);
}

// Gives the slots their rows: mine[b] is the next row of bucket b.
__device__ __forceinline__ void place_slots(const int32_t* ids, int64_t a, int64_t z, int k, int E,
                                            long long offset, int bits, int* mine, const Batch (&kept)[BATCHES],
                                            int32_t* token_of_row, int32_t* row_of_slot) {
    const int lane = threadIdx.x & 63;
    auto put = [&](int64_t s, const Batch& x) {
        const bool live = s + lane < z;
        const int lead = x.same ? __ffsll(x.same) - 1 : 0;
        int at = 0;
        if (live && lane == lead) at = atomicAdd(&mine[x.bucket], __popcll(x.same));
        at = __shfl(at, lead);
        if (live) {
            const int row = at + __popcll(x.same & ((1ull << lane) - 1));
            row_of_slot[s + lane] = row;
            token_of_row[row] = (int32_t)((s + lane) / k);
        }
    };
#pragma unroll
    for (int i = 0; i < BATCHES; ++i)
        if (a + i * 64 < z) put(a + i * 64, kept[i]);
    for (int64_t s = a + BATCHES * 64; s < z; s += 64) {
        Batch x;
        const bool live = s + lane < z;
        x.bucket = live ? bucket_of(ids[s + lane], offset, E) : 0;
        x.same = same_bucket(x.bucket, bits, live);
        put(s, x);
    }
}

// One workgroup. LDS: counts [waves][E + 1], 16 wave sums.
__global__ __launch_bounds__(1024) void sort_small_kernel(const int32_t* __restrict__ ids, int n, int k,
                                                          int E, long long offset, int bits,
                                                          int32_t* __restrict__ offsets,
                                                          int32_t* __restrict__ token_of_row,
                                                          int32_t* __restrict__ row_of_slot) {
    extern __shared__ int smem[];
    const int wave = threadIdx.x >> 6, waves = blockDim.x >> 6;
    int* counts = smem;
    int* tmp = counts + waves * (E + 1);
    for (int i = threadIdx.x; i < waves * (E + 1); i += blockDim.x) counts[i] = 0;
    __syncthreads();
    const int64_t per = ((n + waves - 1) / waves + 63) / 64 * 64;
    const int64_t a = wave * per, z = min(a + per, (int64_t)n);
    Batch kept[BATCHES];
    count_slots(ids, a, z, E, offset, bits, counts + wave * (E + 1), kept);
    __syncthreads();
    int before = 0;
    for (int b0 = 0; b0 <= E; b0 += blockDim.x) {
        const int b = b0 + threadIdx.x;
        int mine = 0, total;
        if (b <= E)
            for (int w = 0; w < waves; ++w) mine += counts[w * (E + 1) + b];
        int at = before + block_scan(mine, tmp, &total);
        if (b <= E) {
            offsets[b] = at;  // [E]: where the other shards' slots start
            for (int w = 0; w < waves; ++w) {
                const int c = counts[w * (E + 1) + b];
                counts[w * (E + 1) + b] = at;
                at += c;
            }
        }
        before += total;
    }
    __syncthreads();
    place_slots(ids, a, z, k, E, offset, bits, counts + wave * (E + 1), kept, token_of_row, row_of_slot);
}

__global__ __launch_bounds__(512) void sort_count_kernel(const int32_t* __restrict__ ids, int64_t n,
                                                         int64_t len, int E, long long offset,
                                                         int32_t* __restrict__ chunk_counts) {
    extern __shared__ int smem[];
    for (int i = threadIdx.x; i <= E; i += blockDim.x) smem[i] = 0;
    __syncthreads();
    const int64_t a = blockIdx.x * len, z = min(a + len, n);
    for (int64_t s = a + threadIdx.x; s < z; s += blockDim.x)
        atomicAdd(&smem[bucket_of(ids[s], offset, E)], 1);
    __syncthreads();
    for (int i = threadIdx.x; i <= E; i += blockDim.x) chunk_counts[(int64_t)blockIdx.x * (E + 1) + i] = smem[i];
}

__global__ __launch_bounds__(512) void sort_place_kernel(const int32_t* __restrict__ ids, int64_t n,
                                                         int64_t len, int k, int E, long long offset,
                                                         int bits, const int32_t* __restrict__ chunk_counts,
                                                         int32_t* __restrict__ offsets,
                                                         int32_t* __restrict__ token_of_row,
                                                         int32_t* __restrict__ row_of_slot) {
    extern __shared__ int smem[];
    const int wave = threadIdx.x >> 6, waves = blockDim.x >> 6;
    int* counts = smem;
    int* tmp = counts + waves * (E + 1);
    for (int i = threadIdx.x; i < waves * (E + 1); i += blockDim.x) counts[i] = 0;
    __syncthreads();
    const int64_t first = blockIdx.x * len, last = min(first + len, n);
    const int64_t per = ((last - first + waves - 1) / waves + 63) / 64 * 64;
    const int64_t a = first + wave * per, z = min(a + per, last);
    Batch kept[BATCHES];
    count_slots(ids, a, z, E, offset, bits, counts + wave * (E + 1), kept);
    __syncthreads();
    int before = 0;  // rows of the buckets below this step's
    for (int b0 = 0; b0 <= E; b0 += blockDim.x) {
        const int b = b0 + threadIdx.x;
        int prior = 0, all = 0;
        if (b <= E) {
#pragma unroll 16
            for (int c = 0; c < (int)gridDim.x; ++c) {
                const int v = chunk_counts[(int64_t)c * (E + 1) + b];
                if (c < (int)blockIdx.x) prior += v;
                all += v;
            }
        }
        int total;
        int at = before + block_scan(all, tmp, &total);
        if (b <= E) {
            if (blockIdx.x == 0) offsets[b] = at;
            at += prior;
            for (int w = 0; w < waves; ++w) {
                const int c = counts[w * (E + 1) + b];
                counts[w * (E + 1) + b] = at;
                at += c;
            }
        }
        before += total;
    }
    __syncthreads();
    place_slots(ids, a, z, k, E, offset, bits, counts + wave * (E + 1), kept, token_of_row, row_of_slot);
}

hipError_t launch_sort(const int32_t* ids, int64_t T, int k, int E, int64_t offset, int32_t* offsets,
                       int32_t* token_of_row, int32_t* row_of_slot, int32_t* counts, hipStream_t s) {
    const int64_t n = T * k;
    int bits = 0;
    while ((E >> bits) != 0) ++bits;
    const int64_t chunks = sort_chunks(n);
    if (chunks == 0) {
        // a wave per 64 slots, enough threads to scan the buckets, LDS within 64 KB
        int waves = (int)((n + 63) / 64), scan = (E + 63) / 64;
        if (scan > 4) scan = 4;
        if (waves < scan) waves = scan;
        const int most = (int)((65536 - 64) / sizeof(int)) / (E + 1);
        if (waves > most) waves = most;
        if (waves > 16) waves = 16;
        const size_t lds = ((size_t)waves * (E + 1) + 16) * sizeof(int);
        hipLaunchKernelGGL(sort_small_kernel, dim3(1), dim3(64 * waves), lds, s, ids, (int)n, k, E,
                           (long long)offset, bits, offsets, token_of_row, row_of_slot);
        return hipGetLastError();
    }
    const int64_t len = chunk_len(n);
    hipLaunchKernelGGL(sort_count_kernel, dim3((unsigned)chunks), dim3(512), (E + 1) * sizeof(int), s, ids,
                       n, len, E, (long long)offset, counts);
    const size_t lds = ((size_t)8 * (E + 1) + 16) * sizeof(int);
    hipLaunchKernelGGL(sort_place_kernel, dim3((unsigned)chunks), dim3(512), lds, s, ids, n, len, k, E,
                       (long long)offset, bits, counts, offsets, token_of_row, row_of_slot);
    return hipGetLastError();
}

}  // namespace miexp
