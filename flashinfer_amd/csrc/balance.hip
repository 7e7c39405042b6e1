// The balance loss of a router and the slots of each expert (mi_layer_balance),
// and the gradient of its logits.
//
//   P[t, :] = softmax(l) or sigma(l) / sum sigma(l),  Pbar_s = sum_t P / n_s
//   loss = 1/S' sum_s sum_e f_se Pbar_se,  f_se = E c_se / (k n_s)
//   dl_j = g P_j (w_j - sum_e P_e w_e) (times 1 - sigma_j for the sigmoids),
//   w_e = f_se / (n_s S') = dloss / dP_e
//
// Tokens go in chunks, and a piece is what one sequence has of one chunk: piece
// number s + chunk rises along the batch, so the sequence of a piece is found
// by bisection over g(s) = s + first(s) / chunk, and there are at most S +
// chunks of them, whatever the lengths. A workgroup sums the probabilities and
// counts the slots of its piece; a second launch sums the pieces of each
// sequence, in columns of experts where there are many; a third the columns and
// the sequences, where there are more than one. All sums are in a fixed order;
// the only atomics count whole numbers.
//
// 65536 x 256 in fp32 with sigmoids: pieces 19 us (3.6 TB/s), their sums 9 and 3,
// gradient 24 (5.7 TB/s: a read and a write of 67 MB). A wave keeps up to four
// tokens on their way; exponentials and quotients are the hardware's with one
// correction, sums over lanes go by DPP. 64 x 256: 4.4, 4 and 3.5 us, all latency;
// there a training step takes what autograd takes on the host, 53 us.
#include "layer_common.hpp"

namespace miexp {

struct BalanceCall {
    const void* logits;
    const int32_t* ids;
    const int32_t* offsets;
    const uint8_t* mask;
    float* loss;
    int32_t* counts;
    float* weights;
    float* part;        // [pieces, E] sums of P
    int32_t* part_n;    // [pieces, E + 1] slots, and tokens that count
    float* seq_loss;    // [S, columns]
    int32_t* some;      // [S] whether the sequence has a token that counts
    int64_t T, S, stride;
    int E, k, chunk, sigmoid;
    int columns;        // workgroups of the second launch for a sequence
    int64_t pieces;
};

// First token of sequence s, and of s + 1 its end: clamped and non-decreasing
// from one to the next.
__device__ __forceinline__ int64_t bound(const BalanceCall& p, int64_t s) {
    if (!p.offsets) return s ? p.T : 0;
    return max((int64_t)0, min((int64_t)p.offsets[s], p.T));
}

// The sequence of token t: the last one that starts at or before it, if t is
// inside; -1 for a token of none.
__device__ __forceinline__ int64_t sequence_of(const BalanceCall& p, int64_t t) {
    if (!p.offsets) return 0;
    int64_t lo = 0, hi = p.S;  // bound(lo) <= t < bound(hi), if it is inside at all
    if (t < bound(p, 0) || t >= bound(p, p.S)) return -1;
    while (hi - lo > 1) {
        const int64_t mid = (lo + hi) >> 1;
        if (bound(p, mid) <= t) lo = mid; else hi = mid;
    }
    return lo;
}

// v of the lane that a DPP control names, in every lane (all lanes are there).
template <int CTRL>
__device__ __forceinline__ float dpp(float v) {
    return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, 0xf, 0xf, true));
}

// f over groups of TX lanes, the same bits in each of them: pairs within 4
// lanes, mirrored halves of 8 and 16, rows of 16 exchanged.
template <int TX, class F>
__device__ __forceinline__ float over_lanes(float a, F f) {
    a = f(a, dpp<0xb1>(a));   // quad_perm 1 0 3 2
    a = f(a, dpp<0x4e>(a));   // quad_perm 2 3 0 1
    a = f(a, dpp<0x141>(a));  // row_half_mirror
    if constexpr (TX >= 16) a = f(a, dpp<0x140>(a));  // row_mirror
    if constexpr (TX >= 32) {
        const auto s = __builtin_amdgcn_permlane16_swap(__float_as_uint(a), __float_as_uint(a), false, false);
        a = f(__uint_as_float(s[0]), __uint_as_float(s[1]));
    }
    if constexpr (TX >= 64) {
        const auto s = __builtin_amdgcn_permlane32_swap(__float_as_uint(a), __float_as_uint(a), false, false);
        a = f(__uint_as_float(s[0]), __uint_as_float(s[1]));
    }
    return a;
}

// e^a = 2^(hi + lo) with hi + lo = a log2(e) to twice the precision; past 87
// (2^125.5) in the precision of hi alone, below 2^-126 zero.
__device__ __forceinline__ float exp_of(float a) {
    constexpr float L2E = 1.44269502f, L2E_LO = 1.92596299e-8f, LN2 = 0.693147182f;
    const float hi = a * L2E, lo = fmaf(a, L2E_LO, fmaf(a, L2E, -hi));
    const float x = __builtin_amdgcn_exp2f(hi);
    return fabsf(a) < 87.f ? fmaf(x, lo * LN2, x) : x;
}

// A wave's TX lanes hold a token's logits: lane j of them V at a time from j V,
// STEPS times. Rows end where E does: lanes past it hold -inf.
template <class T, int V, int STEPS, int TX>
struct Row {
    float x[STEPS][V];

    __device__ __forceinline__ static int at(int i) { return (i * TX + (threadIdx.x & (TX - 1))) * V; }

    __device__ __forceinline__ void load_row(const T* row, int E) {
#pragma unroll
        for (int i = 0; i < STEPS; ++i) {
            if (at(i) + V <= E) {
                load<T, V>(row + at(i), x[i]);
            } else {
#pragma unroll
                for (int v = 0; v < V; ++v) x[i][v] = at(i) + v < E ? (float)row[at(i) + v] : -INFINITY;
            }
        }
    }
    __device__ __forceinline__ static float sum(float a) {
        return over_lanes<TX>(a, [](float b, float c) { return b + c; });
    }
    __device__ __forceinline__ static float largest(float a) {
        return over_lanes<TX>(a, [](float b, float c) { return fmaxf(b, c); });
    }
    // x becomes P; `slope` 1 for the softmax, 1 - sigma for the sigmoids.
    template <bool SLOPE>
    __device__ __forceinline__ void scores(bool sigmoid, float (&slope)[STEPS][V]) {
        float total = 0.f;
        if (sigmoid) {
            float l[STEPS][V];
#pragma unroll
            for (int i = 0; i < STEPS; ++i)
#pragma unroll
                for (int v = 0; v < V; ++v) {
                    l[i][v] = x[i][v];
                    const float e = exp_of(-x[i][v]);
                    const float d = 1.f + e, rc = __builtin_amdgcn_rcpf(d);
                    // past 2^126 the reciprocal is 0, and so is such a score beside a sum of 1e-8
                    const bool near = d < 8e37f;
                    const float s = near ? fmaf(fmaf(-rc, d, 1.f), rc, rc) : rc;
                    // 1 - sigma without cancellation
                    if constexpr (SLOPE) slope[i][v] = near ? e * s : 1.f;
                    x[i][v] = s;
                    total += s;
                }
            // Scores so low that their sigmoids are e^l in fp32: quotients of e^(l - top), which stay in range.
            if (sum(total) < 1e-8f) {
                float top = -INFINITY;
#pragma unroll
                for (int i = 0; i < STEPS; ++i)
#pragma unroll
                    for (int v = 0; v < V; ++v) top = fmaxf(top, l[i][v]);
                top = largest(top);
                if (top == -INFINITY) top = 0.f;
                total = 0.f;
#pragma unroll
                for (int i = 0; i < STEPS; ++i)
#pragma unroll
                    for (int v = 0; v < V; ++v) {
                        x[i][v] = exp_of(l[i][v] - top);
                        total += x[i][v];
                    }
            }
        } else {
            float top = -INFINITY;
#pragma unroll
            for (int i = 0; i < STEPS; ++i)
#pragma unroll
                for (int v = 0; v < V; ++v) top = fmaxf(top, x[i][v]);
            top = largest(top);
            if (top == -INFINITY) top = 0.f;  // a row of them: zeros, whatever they are divided by
#pragma unroll
            for (int i = 0; i < STEPS; ++i)
#pragma unroll
                for (int v = 0; v < V; ++v) {
                    if constexpr (SLOPE) slope[i][v] = 1.f;
                    x[i][v] = exp_of(x[i][v] - top);
                    total += x[i][v];
                }
        }
        total = sum(total);
        const float r = total == 0.f ? 0.f : 1.f / total;
#pragma unroll
        for (int i = 0; i < STEPS; ++i)
#pragma unroll
            for (int v = 0; v < V; ++v) x[i][v] *= r;
    }
};

// Sums of one piece by WAVES waves. LDS: sums [min(WAVES, 8)][E], counts [E + 1].
template <class T, int V, int STEPS, int TX, int WAVES>
__global__ __launch_bounds__(64 * WAVES) void balance_piece_kernel(BalanceCall p) {
    extern __shared__ float smem[];
    constexpr int PER = 64 / TX, HALF = WAVES > 8 ? 8 : WAVES;  // PER: tokens of a wave at a time
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    float* sums = smem;
    int* counts = reinterpret_cast<int*>(smem + HALF * p.E);
    // the last s with s + first(s) / chunk <= piece
    const int64_t piece = blockIdx.x;
    int64_t s = 0, hi = p.S;
    while (hi - s > 1) {
        const int64_t mid = (s + hi) >> 1;
        if (mid + bound(p, mid) / p.chunk <= piece) s = mid; else hi = mid;
    }
    const int64_t c = piece - s;
    const int64_t a = max(bound(p, s), c * p.chunk), z = min(bound(p, s + 1), (c + 1) * p.chunk);
    for (int i = threadIdx.x; i <= p.E; i += 64 * WAVES) counts[i] = 0;
    __syncthreads();
    typedef Row<T, V, STEPS, TX> R;
    constexpr int U = 16 / (STEPS * V) > 4 ? 4 : 16 / (STEPS * V);  // tokens on their way
    float acc[STEPS][V] = {};
    int mine = 0;  // tokens that count
    for (int64_t t0 = a + wave * PER; t0 < z; t0 += WAVES * PER * U) {
        R row[U];
        bool live[U];
        int id[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int64_t t = t0 + u * WAVES * PER + lane / TX;
            live[u] = t < z && (!p.mask || p.mask[t]);
            const int64_t from = live[u] ? t : t0;
            row[u].load_row((const T*)p.logits + from * p.stride, p.E);
            const int j = lane & (TX - 1);
            id[u] = live[u] && j < p.k ? p.ids[from * p.k + j] : -1;
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            float none[STEPS][V];
            row[u].template scores<false>(p.sigmoid, none);
            if (!live[u]) continue;
            ++mine;
#pragma unroll
            for (int i = 0; i < STEPS; ++i)
#pragma unroll
                for (int v = 0; v < V; ++v) acc[i][v] += row[u].x[i][v];
            if (id[u] >= 0 && id[u] < p.E) atomicAdd(&counts[id[u]], 1);
            if (TX < MI_LAYER_MAX_TOP_K && p.k > TX) {
                const int64_t t = t0 + u * WAVES * PER + lane / TX;
                for (int j = (lane & (TX - 1)) + TX; j < p.k; j += TX) {
                    const int e = p.ids[t * p.k + j];
                    if (e >= 0 && e < p.E) atomicAdd(&counts[e], 1);
                }
            }
        }
    }
    // the wave's tokens side by side, then the waves: the last eight of 16 to the first ones
#pragma unroll
    for (int i = 0; i < STEPS; ++i)
#pragma unroll
        for (int v = 0; v < V; ++v)
#pragma unroll
            for (int d = TX; d < 64; d <<= 1) acc[i][v] += __shfl_xor(acc[i][v], d);
    if ((lane & (TX - 1)) == 0 && mine) atomicAdd(&counts[p.E], mine);
    auto each = [&](bool mine, auto f) {
        if (!mine || lane >= TX) return;
        float* row = sums + (wave % HALF) * p.E;
#pragma unroll
        for (int i = 0; i < STEPS; ++i)
#pragma unroll
            for (int v = 0; v < V; ++v)
                if (R::at(i) + v < p.E) f(row[R::at(i) + v], acc[i][v]);
    };
    if constexpr (WAVES > HALF) {
        each(wave >= HALF, [](float& at, float& a) { at = a; });
        __syncthreads();
        each(wave < HALF, [](float& at, float& a) { at += a; });
    } else {
        each(true, [](float& at, float& a) { at = a; });
    }
    __syncthreads();
    for (int e = threadIdx.x; e < p.E; e += 64 * WAVES) {
        float all = 0.f;
#pragma unroll
        for (int w = 0; w < HALF; ++w) all += sums[w * p.E + e];
        p.part[piece * p.E + e] = all;
    }
    for (int e = threadIdx.x; e <= p.E; e += 64 * WAVES) p.part_n[piece * (p.E + 1) + e] = counts[e];
}

// Sum over a workgroup of 1024 threads of one value each, in a fixed order.
__device__ __forceinline__ float block_sum(float v, float* tmp) {
#pragma unroll
    for (int d = 32; d >= 1; d >>= 1) v += __shfl_xor(v, d);
    if ((threadIdx.x & 63) == 0) tmp[threadIdx.x >> 6] = v;
    __syncthreads();
    float all = 0.f;
    for (int w = 0; w < (int)(blockDim.x >> 6); ++w) all += tmp[w];
    __syncthreads();
    return all;
}

// Sums the pieces of sequence blockIdx.x / p.columns, of its columns of experts
// (all of them in turn if p.columns is 1): COLUMNS threads side by side take
// the experts, 1024 / COLUMNS rows of them the pieces.
template <int COLUMNS>
__global__ __launch_bounds__(1024) void balance_sum_kernel(BalanceCall p) {
    constexpr int ROWS = 1024 / COLUMNS;
    __shared__ float sum[1024], tmp[16];
    __shared__ int num[1024];
    const int64_t s = blockIdx.x / p.columns, a = bound(p, s), z = bound(p, s + 1);
    const int part = (int)(blockIdx.x - s * p.columns);
    const int64_t first = s + a / p.chunk, end = z > a ? s + (z - 1) / p.chunk + 1 : first;
    const int col = threadIdx.x % COLUMNS, row = threadIdx.x / COLUMNS;
    int n = 0;
    for (int64_t i = first + threadIdx.x; i < end; i += 1024) n += p.part_n[i * (p.E + 1) + p.E];
#pragma unroll
    for (int d = 32; d >= 1; d >>= 1) n += __shfl_xor(n, d);
    if ((threadIdx.x & 63) == 0) num[threadIdx.x >> 6] = n;
    __syncthreads();
    n = 0;
#pragma unroll
    for (int w = 0; w < 16; ++w) n += num[w];
    __syncthreads();
    const float share = n ? 1.f / (float)n : 0.f, unit = share * (float)p.E / (float)p.k;
    float loss = 0.f;
    for (int e0 = part * COLUMNS; e0 < p.E; e0 += COLUMNS * p.columns) {
        const int e = e0 + col;
        float x = 0.f;
        int c = 0;
        if (e < p.E) {
#pragma unroll 4
            for (int64_t i = first + row; i < end; i += ROWS) {
                x += p.part[i * p.E + e];
                c += p.part_n[i * (p.E + 1) + e];
            }
        }
        sum[threadIdx.x] = x;
        num[threadIdx.x] = c;
        __syncthreads();
        if (row == 0 && e < p.E) {
#pragma unroll 8
            for (int r = 1; r < ROWS; ++r) {
                x += sum[r * COLUMNS + col];
                c += num[r * COLUMNS + col];
            }
            const float w = (float)c * unit * share;
            p.counts[s * p.E + e] = c;
            p.weights[s * p.E + e] = w;
            loss += w * x;
        }
        __syncthreads();
    }
    loss = block_sum(loss, tmp);
    if (threadIdx.x) return;
    if (p.S == 1 && p.columns == 1) {
        p.loss[0] = loss;
    } else {
        p.seq_loss[blockIdx.x] = loss;
        if (part == 0) p.some[s] = n > 0;
    }
}

// The mean over the sequences that have a token, and its share in each weight.
__global__ __launch_bounds__(1024) void balance_mean_kernel(BalanceCall p) {
    __shared__ float tmp[16];
    float loss = 0.f, some = 0.f;
    for (int64_t i = threadIdx.x; i < p.S * p.columns; i += 1024) loss += p.seq_loss[i];
    for (int64_t s = threadIdx.x; s < p.S; s += 1024) some += (float)p.some[s];  // whole numbers, exact up to 2^24
    some = block_sum(some, tmp);
    const float share = some > 0.f ? 1.f / some : 0.f;
    if (blockIdx.x == 0) {
        loss = block_sum(loss, tmp) * share;
        if (threadIdx.x == 0) p.loss[0] = loss;
    }
    if (p.S == 1) return;
    for (int64_t i = (int64_t)blockIdx.x * 1024 + threadIdx.x; i < p.S * p.E; i += (int64_t)gridDim.x * 1024)
        p.weights[i] *= share;
}

// SEQS: tokens look up their sequence and its weights; else all have the same,
// which stay in registers.
template <class T, int V, int STEPS, int TX, bool SEQS>
__global__ __launch_bounds__(256) void balance_backward_kernel(BalanceCall p, const float* __restrict__ grad_loss,
                                                               T* __restrict__ grad, int64_t grad_stride) {
    constexpr int PER = 64 / TX, U = STEPS * V > 4 ? 1 : 2;  // tokens on their way
    const int lane = threadIdx.x & 63;
    const float g = *grad_loss;
    typedef Row<T, V, STEPS, TX> R;
    float w[STEPS][V];
    auto weights_of = [&](int64_t s) __attribute__((always_inline)) {
        const float* from = p.weights + s * p.E;
#pragma unroll
        for (int i = 0; i < STEPS; ++i)
#pragma unroll
            for (int v = 0; v < V; ++v) w[i][v] = R::at(i) + v < p.E ? from[R::at(i) + v] : 0.f;
    };
    if constexpr (!SEQS) weights_of(0);
    const int64_t step = (int64_t)gridDim.x * 4 * PER;
    for (int64_t t0 = ((int64_t)blockIdx.x * 4 + (threadIdx.x >> 6)) * PER; t0 < p.T; t0 += step * U) {
        R row[U];
#pragma unroll
        for (int u = 0; u < U; ++u)
            row[u].load_row((const T*)p.logits + min(t0 + u * step + lane / TX, p.T - 1) * p.stride, p.E);
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int64_t t = t0 + u * step + lane / TX, from = min(t, p.T - 1);
            bool out = p.mask && !p.mask[from];
            if constexpr (SEQS) {
                const int64_t s = sequence_of(p, from);
                weights_of(max(s, (int64_t)0));
                out |= s < 0;
            }
            float slope[STEPS][V];
            row[u].template scores<true>(p.sigmoid, slope);
            float dot = 0.f;
#pragma unroll
            for (int i = 0; i < STEPS; ++i)
#pragma unroll
                for (int v = 0; v < V; ++v) dot = fmaf(row[u].x[i][v], w[i][v], dot);
            dot = R::sum(dot);
            if (t >= p.T) continue;
            T* to = grad + t * grad_stride;
#pragma unroll
            for (int i = 0; i < STEPS; ++i) {
                float d[V];
#pragma unroll
                for (int v = 0; v < V; ++v)
                    d[v] = out ? 0.f : g * (row[u].x[i][v] * slope[i][v] * (w[i][v] - dot));
                if (R::at(i) + V <= p.E) {
                    store<T, V>(to + R::at(i), d);
                } else {
#pragma unroll
                    for (int v = 0; v < V; ++v)
                        if (R::at(i) + v < p.E) to[R::at(i) + v] = (T)d[v];
                }
            }
        }
    }
}

// Tokens of a chunk: 16 for four waves up to 4096 tokens, where latency counts;
// then 64 or more for 16 waves, at most 512 chunks, two workgroups for each CU
// (65536 x 256 in fp32: 18 us for the pieces and 21 for their sums with 2048
// chunks of 32).
constexpr int BALANCE_SHORT = 16;
int balance_chunk(int64_t T) {
    if (T <= 4096) return BALANCE_SHORT;
    int64_t chunk = 64;
    while (chunk * 512 < T) chunk *= 2;
    return (int)chunk;
}
// Workgroups that sum a sequence's pieces: one, or one for 16 experts where that
// takes off more than a launch that joins them (which several sequences need anyway).
int balance_columns(int64_t T, int64_t S, int E) {
    const int64_t pieces = T / balance_chunk(T) / S;
    return pieces > (S > 1 ? 4 : 32) ? (E + 15) / 16 : 1;
}
int64_t balance_pieces(int64_t T, int64_t S) {
    const int chunk = balance_chunk(T);
    return S + (T + chunk - 1) / chunk;
}

struct BalanceSpace {
    size_t part, part_n, seq_loss, some, total;
};
BalanceSpace balance_space(int64_t T, int64_t S, int E) {
    auto up = [](size_t v) { return (v + 255) / 256 * 256; };
    const size_t pieces = (size_t)balance_pieces(T, S);
    BalanceSpace b;
    b.part = 0;
    b.part_n = up(b.part + pieces * E * 4);
    b.seq_loss = up(b.part_n + pieces * (E + 1) * 4);
    b.some = up(b.seq_loss + (size_t)S * balance_columns(T, S, E) * 4);
    b.total = up(b.some + (size_t)S * 4);
    return b;
}
size_t balance_workspace(int64_t T, int64_t S, int E) { return balance_space(T, S, E).total; }

BalanceCall balance_call(const mi_layer_balance_args& a) {
    BalanceCall p{};
    p.logits = a.logits;
    p.ids = a.topk_ids;
    p.offsets = a.seq_offsets;
    p.mask = a.mask;
    p.loss = a.loss;
    p.counts = a.counts;
    p.weights = a.weights;
    p.T = a.num_tokens;
    p.S = a.num_seqs;
    p.stride = a.logits_stride;
    p.E = a.num_experts;
    p.k = a.top_k;
    p.chunk = balance_chunk(a.num_tokens);
    p.columns = balance_columns(a.num_tokens, a.num_seqs, a.num_experts);
    p.sigmoid = a.score == MI_LAYER_SCORE_SIGMOID;
    p.pieces = balance_pieces(a.num_tokens, a.num_seqs);
    return p;
}

// Calls f with the form of a row: V values of a lane at a time (16 bytes, where
// the rows are aligned to that), STEPS of them, TX lanes.
template <class T, class F>
hipError_t by_row(int E, bool vec, F f) {
    constexpr int W = 16 / (int)sizeof(T);
    if (vec) {
        if (E <= 8 * W) return f(IntC<W>{}, IntC<1>{}, IntC<8>{});
        if (E <= 16 * W) return f(IntC<W>{}, IntC<1>{}, IntC<16>{});
        if (E <= 32 * W) return f(IntC<W>{}, IntC<1>{}, IntC<32>{});
        if (E <= 64 * W) return f(IntC<W>{}, IntC<1>{}, IntC<64>{});
        return f(IntC<W>{}, IntC<1024 / (64 * W)>{}, IntC<64>{});
    }
    if (E <= 64) return f(IntC<1>{}, IntC<1>{}, IntC<64>{});
    if (E <= 256) return f(IntC<1>{}, IntC<4>{}, IntC<64>{});
    return f(IntC<1>{}, IntC<16>{}, IntC<64>{});
}
template <class F>
hipError_t by_type(int dtype, F f) {
    if (dtype == MI_LAYER_F32) return f(float{});
    if (dtype == MI_LAYER_F16) return f(_Float16{});
    return f(__bf16{});
}
template <class T>
bool balance_vec(const mi_layer_balance_args& a) {
    return (uint64_t)a.logits % 16 == 0 && a.logits_stride % (16 / (int)sizeof(T)) == 0;
}

hipError_t launch_balance(const mi_layer_balance_args& a, hipStream_t s) {
    BalanceCall p = balance_call(a);
    const BalanceSpace b = balance_space(a.num_tokens, a.num_seqs, a.num_experts);
    uint8_t* ws = (uint8_t*)a.workspace;
    p.part = (float*)(ws + b.part);
    p.part_n = (int32_t*)(ws + b.part_n);
    p.seq_loss = (float*)(ws + b.seq_loss);
    p.some = (int32_t*)(ws + b.some);
    hipError_t e = by_type(a.dtype, [&](auto t) {
        typedef decltype(t) T;
        return by_row<T>(a.num_experts, balance_vec<T>(a), [&](auto v, auto steps, auto tx) {
            constexpr int V = decltype(v)::value, STEPS = decltype(steps)::value, TX = decltype(tx)::value;
            const dim3 grid((unsigned)p.pieces);
            if (p.chunk == BALANCE_SHORT)
                hipLaunchKernelGGL((balance_piece_kernel<T, V, STEPS, TX, 4>), grid, dim3(256),
                                   (size_t)(5 * p.E + 1) * 4, s, p);
            else
                hipLaunchKernelGGL((balance_piece_kernel<T, V, STEPS, TX, 16>), grid, dim3(1024),
                                   (size_t)(9 * p.E + 1) * 4, s, p);
            return hipGetLastError();
        });
    });
    if (e != hipSuccess) return e;
    if (p.columns > 1)
        hipLaunchKernelGGL(balance_sum_kernel<16>, dim3((unsigned)(p.S * p.columns)), dim3(1024), 0, s, p);
    else if (p.E <= 64)
        hipLaunchKernelGGL(balance_sum_kernel<64>, dim3((unsigned)p.S), dim3(1024), 0, s, p);
    else
        hipLaunchKernelGGL(balance_sum_kernel<256>, dim3((unsigned)p.S), dim3(1024), 0, s, p);
    e = hipGetLastError();
    if (e != hipSuccess || (p.S == 1 && p.columns == 1)) return e;
    const int64_t blocks = p.S == 1 ? 1 : (p.S * p.E + 1023) / 1024;
    hipLaunchKernelGGL(balance_mean_kernel, dim3((unsigned)(blocks < 256 ? blocks : 256)), dim3(1024), 0, s, p);
    return hipGetLastError();
}

hipError_t launch_balance_backward(const mi_layer_balance_args& a, const float* grad_loss, void* grad,
                                   int64_t grad_stride, hipStream_t s) {
    const BalanceCall p = balance_call(a);
    return by_type(a.dtype, [&](auto t) {
        typedef decltype(t) T;
        const bool vec = balance_vec<T>(a) && (uint64_t)grad % 16 == 0 && grad_stride % (16 / (int)sizeof(T)) == 0;
        return by_row<T>(a.num_experts, vec, [&](auto v, auto steps, auto tx) {
            constexpr int TX = decltype(tx)::value;
            // 8 workgroups for each CU go over the tokens
            const int64_t blocks = (p.T + 4 * (64 / TX) - 1) / (4 * (64 / TX));
            const dim3 grid((unsigned)(blocks < 2048 ? blocks : 2048));
            auto launch = [&](auto kernel) {
                hipLaunchKernelGGL(kernel, grid, dim3(256), 0, s, p, grad_loss, (T*)grad, grad_stride);
                return hipGetLastError();
            };
            constexpr int VV = decltype(v)::value, ST = decltype(steps)::value;
            return p.offsets ? launch(balance_backward_kernel<T, VV, ST, TX, true>)
                             : launch(balance_backward_kernel<T, VV, ST, TX, false>);
        });
    });
}

}  // namespace miexp
