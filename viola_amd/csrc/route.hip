// A router's choice of experts with its gates, places and counts, the balance loss, and their gradient.
//
// Scores u (up to one factor for a row): u_e = exp(l_e - m) for softmax, sigmoid(l_e) / sigmoid(m) for sigmoid, with m the row's largest
// logit, so a row far from zero neither overflows nor vanishes. p = u / sum u.
//
//   choice    the top_k largest logits, NaN above all numbers, ties to the lowest index, -inf never
//   gates     scale u_i / (sum over the chosen), or scale p_i (softmax) / scale sigmoid(l_i)
//   balance   mean over sequences of E sum_e (c_e / (n k)) (sum_t p_te / n), with c_e choices of e in its n counted tokens
//   position  (choices of experts before e) + (choices of e by tokens before t): rows sorted by expert, then by token
//   gradient  dl_te = slope (p_te (C_e - sum_j p_tj C_j) + the gates' part), C_e = E c_e / (n^2 k sequences) times the loss's gradient,
//             slope = 1 (softmax) or 1 - sigmoid(l) (sigmoid)
//
// A token that the mask leaves out, or whose logits are all -inf, is not counted, chooses nothing and has no gradient.
//
// A row belongs to `LANES` lanes of VALUES logits each; a block takes a run of tokens (a portion) of one sequence. Counts are integers
// and probabilities are added in one order, so results do not change from run to run: places of equal experts come from a bit for
// each token in LDS, blocks leave their counts and sums behind, and a second kernel adds those of the blocks before.
#include "block_ops.hpp"

#include <type_traits>

using namespace viola;

namespace {

constexpr int THREADS = 512, MOST_EXPERTS = 1024, MOST_CHOSEN = 32, MOST_BLOCKS = 256;

struct RouteArgs {
    const void* logits;
    int64_t pitch, tokens;
    int dtype, experts, top_k, sigmoid, normalize, whole;                    // whole: rows can be read four logits at a time
    float scale;
    const uint8_t* mask;
    int64_t sequence, sequences, per_sequence, chunk, portions, per_block, blocks;
    // choices made elsewhere (balance alone)
    const void* given;
    int given_wide;
    // results
    int *chosen, *positions, *counts, *offsets;
    float *gates, *loss, *cost;                                              // cost: [sequences][experts], E c / (n^2 k sequences)
    float2* stats;                                                           // m, 1 / sum u of a row; 1 / sum u = 0: not counted
    // left behind by the blocks
    int *block_counts, *portion_counts, *portion_tokens;
    float* portion_sums;
};

// ---------------------------------------------------------------------------------------------------- over the lanes of a row
template <int CTRL> __device__ __forceinline__ uint32_t dpp(uint32_t v) { return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xf, 0xf, true); }

template <int LANES, typename F> __device__ __forceinline__ uint32_t over_lanes(uint32_t v, F&& f) {
    if constexpr (LANES >= 2) v = f(v, dpp<0xB1>(v));
    if constexpr (LANES >= 4) v = f(v, dpp<0x4E>(v));
    if constexpr (LANES >= 8) v = f(v, dpp<0x141>(v));                       // halves of eight hold one value each: a mirror swaps them
    if constexpr (LANES >= 16) v = f(v, dpp<0x140>(v));
    if constexpr (LANES >= 32) v = f(v, (uint32_t)__shfl_xor((int)v, 16, WAVE));
    if constexpr (LANES >= 64) v = f(v, (uint32_t)__shfl_xor((int)v, 32, WAVE));
    return v;
}
template <int LANES> __device__ __forceinline__ uint32_t lanes_max(uint32_t v) { return over_lanes<LANES>(v, [](uint32_t a, uint32_t b) { return a > b ? a : b; }); }
template <int LANES> __device__ __forceinline__ uint32_t lanes_min(uint32_t v) { return over_lanes<LANES>(v, [](uint32_t a, uint32_t b) { return a < b ? a : b; }); }
template <int LANES> __device__ __forceinline__ float lanes_sum(float v) {
    return __uint_as_float(over_lanes<LANES>(__float_as_uint(v), [](uint32_t a, uint32_t b) { return __float_as_uint(__uint_as_float(a) + __uint_as_float(b)); }));
}

// ---------------------------------------------------------------------------------------------------- values
// Order of logits as that of unsigned integers: NaN above all, -0 equal to 0, 0 for -inf, which is never chosen.
__device__ __forceinline__ uint32_t key_of(float l) {
    if (l != l) return 0xffffffffu;
    const uint32_t b = __float_as_uint(l + 0.0f);
    if (b == 0xff800000u) return 0;
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float value_of(uint32_t key) { return __uint_as_float(key & 0x80000000u ? key ^ 0x80000000u : ~key); }

// exp(x) within 2 ulp for x <= 0 (0 below -150): exp2 of the product's two halves, the low one multiplied in afterwards.
__device__ __forceinline__ float exp_of(float x) {
    const float t = x * 1.44269502f;                                         // log2(e) = 1.44269502 + 1.92596e-8
    const float low = fmaf(x, 1.92596299e-8f, fmaf(x, 1.44269502f, -t));
    const float e = __builtin_amdgcn_exp2f(t) * fmaf(low, 0.693147182f, 1.0f);
    return x < -150.0f ? 0.0f : e;
}

// u of a logit in a row whose largest is m
__device__ __forceinline__ float score(int sigmoid, float l, float m) {
    if (!sigmoid) return exp_of(l - m);
    const float t = exp_of(-fabsf(l));                                       // sigmoid(l) = exp(min(l, 0)) / (1 + exp(-|l|))
    return exp_of(fminf(l, 0.0f) - fminf(m, 0.0f)) / (1.0f + t);
}
__device__ __forceinline__ float sigmoid_of(float l) {
    const float t = exp_of(-fabsf(l));
    return (l < 0.0f ? t : 1.0f) / (1.0f + t);
}

// VALUES logits of a lane: runs of four, LANES runs apart
template <int LANES> __device__ __forceinline__ int expert_of(int i, int lane) { return ((i / 4) * LANES + lane) * 4 + i % 4; }

template <int LANES, int VALUES> __device__ __forceinline__ void load_logits(const RouteArgs& a, int64_t token, int lane, float (&l)[VALUES]) {
    const int64_t row = token * a.pitch;
#pragma unroll
    for (int i = 0; i < VALUES; i += 4) {
        const int e = expert_of<LANES>(i, lane);
        if (a.whole && e < a.experts) {                                      // experts is a multiple of four here
            if (a.dtype == VIOLA_F32) {
                const float4 v = *reinterpret_cast<const float4*>(static_cast<const float*>(a.logits) + row + e);
                l[i] = v.x; l[i + 1] = v.y; l[i + 2] = v.z; l[i + 3] = v.w;
            } else {
                const uint2 v = *reinterpret_cast<const uint2*>(static_cast<const uint16_t*>(a.logits) + row + e);
                if (a.dtype == VIOLA_BF16) {
                    l[i] = widen16<bf16_t>(v.x & 0xffffu); l[i + 1] = widen16<bf16_t>(v.x >> 16);
                    l[i + 2] = widen16<bf16_t>(v.y & 0xffffu); l[i + 3] = widen16<bf16_t>(v.y >> 16);
                } else {
                    l[i] = widen16<f16_t>(v.x & 0xffffu); l[i + 1] = widen16<f16_t>(v.x >> 16);
                    l[i + 2] = widen16<f16_t>(v.y & 0xffffu); l[i + 3] = widen16<f16_t>(v.y >> 16);
                }
            }
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j) l[i + j] = e + j < a.experts ? load_float(a.logits, row + e + j, a.dtype) : -__builtin_inff();
        }
    }
}

// ---------------------------------------------------------------------------------------------------- after the blocks
// Of all choices: how many of each expert, how many in blocks before `block`, and the exclusive sum over experts; base[e] is the place of
// the first choice of e in this block. Every thread of the block has to call it; total, before, base: [experts] in LDS.
__device__ __forceinline__ void places(const RouteArgs& a, int64_t block, int* total, int* base) {
    for (int e = threadIdx.x; e < a.experts; e += blockDim.x) total[e] = base[e] = 0;
    __syncthreads();
    int wide = 1;
    while (wide < a.experts) wide *= 2;
    const int slices = wide < (int)blockDim.x ? (int)blockDim.x / wide : 1;
    if ((int)threadIdx.x / wide < slices)
        for (int e = threadIdx.x % wide; e < a.experts; e += blockDim.x) {   // blockDim < wide: one slice, several experts for a thread
            int all = 0, before = 0;
            for (int64_t b = threadIdx.x / wide; b < a.blocks; b += slices) {
                const int c = a.block_counts[b * a.experts + e];
                all += c;
                before += b < block ? c : 0;
            }
            atomicAdd(&total[e], all);
            atomicAdd(&base[e], before);
        }
    __syncthreads();
    // exclusive sums by one wavefront: each lane a run of experts, then over the lanes
    if (threadIdx.x < 64) {
        const int run = (a.experts + 63) / 64, first = threadIdx.x * run;
        int sum = 0;
        for (int e = first; e < first + run && e < a.experts; ++e) sum += total[e];
        int inclusive = sum;
        for (int d = 1; d < 64; d *= 2) {
            const int other = __shfl_up(inclusive, d, 64);
            if ((int)threadIdx.x >= d) inclusive += other;
        }
        int at = inclusive - sum;
        for (int e = first; e < first + run && e < a.experts; ++e) {
            base[e] += at;
            if (block == 0) {
                a.counts[e] = total[e];
                if (a.offsets) a.offsets[e] = at;
            }
            at += total[e];
        }
        if (block == 0 && a.offsets && threadIdx.x == 63) a.offsets[a.experts] = inclusive;
    }
    __syncthreads();
}

// The loss and the experts' costs; one block. piece: [2][blockDim] in LDS, tokens: [per_sequence > 1 ? sequences : 0].
__device__ __forceinline__ void balance(const RouteArgs& a, float* piece, int* tokens, float2 (*slots)[16]) {
    const int m = (int)a.per_sequence;
    if (m > 1) {
        for (int s = threadIdx.x; s < a.sequences; s += blockDim.x) tokens[s] = 0;
        __syncthreads();
        for (int64_t p = threadIdx.x; p < a.portions; p += blockDim.x) atomicAdd(&tokens[p / m], a.portion_tokens[p]);
        __syncthreads();
    }
    const int64_t pairs = a.sequences * a.experts;                           // (sequence, expert)
    int64_t wide = 1;
    while (wide < pairs && wide < (int64_t)blockDim.x) wide *= 2;
    const int slices = (int)(blockDim.x / wide), slice = (int)(threadIdx.x / wide);
    float loss = 0.0f;
    for (int64_t first = 0; first < pairs; first += wide) {
        const int64_t pair = first + threadIdx.x % wide, s = pair / a.experts;
        const int e = (int)(pair % a.experts);
        float sum = 0.0f;
        int count = 0;
        if (pair < pairs)
            for (int64_t p = s * m + slice; p < (s + 1) * m; p += slices) {
                sum += a.portion_sums[p * a.experts + e];
                count += a.portion_counts[p * a.experts + e];
            }
        if (slices > 1) {                                                    // pairs fit the block: one pass of this loop
            piece[threadIdx.x] = sum;
            piece[blockDim.x + threadIdx.x] = __int_as_float(count);
            __syncthreads();
            if (slice == 0)
                for (int u = 1; u < slices; ++u) {
                    sum += piece[u * wide + threadIdx.x];
                    count += __float_as_int(piece[blockDim.x + u * wide + threadIdx.x]);
                }
        }
        if (pair < pairs && slice == 0) {
            const float n = (float)(m > 1 ? tokens[s] : a.portion_tokens[s]);
            const float cost = n > 0.0f ? (float)a.experts * (float)count / (n * n * (float)a.top_k * (float)a.sequences) : 0.0f;
            a.cost[pair] = cost;
            loss = fmaf(cost, sum, loss);
        }
    }
    BlockSums sums(slots);
    loss = sums.one(loss);
    if (threadIdx.x == 0) *a.loss = loss;
}

// ---------------------------------------------------------------------------------------------------- forward
// LDS: running counts and counts at the portion's start [experts] each, bits [experts][words], chosen and values [rows * top_k], factors
// [rows], then sums [8][experts] (over the bits and what follows them, once a portion is done)
template <int LANES> __host__ __device__ constexpr int rows_of() { return THREADS / LANES; }
template <int LANES> __host__ __device__ constexpr int words_of() { return (rows_of<LANES>() + 31) / 32; }

template <int LANES> size_t choose_lds(int experts, int top_k, bool given) {
    const size_t rows = rows_of<LANES>();
    const size_t choice = given ? 0 : (size_t)experts * words_of<LANES>() + 2 * rows * top_k + rows;
    const size_t sums = (size_t)(THREADS / 64) * experts, tail = 2 * THREADS + MOST_BLOCKS;     // the tail is that of `balance`
    size_t most = choice > sums ? choice : sums;
    if (most < tail) most = tail;
    return 4 * (2 * (size_t)experts + most);
}

template <int LANES, int VALUES, bool GIVEN> __global__ __launch_bounds__(THREADS) void choose_kernel(RouteArgs a) {
    extern __shared__ int lds[];
    __shared__ int counted_tokens;
    __shared__ float2 slots[2][16];
    constexpr int ROWS = rows_of<LANES>(), WORDS = words_of<LANES>();
    int *counts = lds, *start = lds + a.experts, *rest = lds + 2 * a.experts;
    uint32_t* bits = reinterpret_cast<uint32_t*>(rest);
    int* chosen = rest + a.experts * WORDS;
    float* values = reinterpret_cast<float*>(chosen + ROWS * a.top_k);
    float* factors = values + ROWS * a.top_k;
    float* sums = reinterpret_cast<float*>(rest);
    const int lane = threadIdx.x % LANES, slot = threadIdx.x / LANES;
    for (int e = threadIdx.x; e < a.experts; e += THREADS) counts[e] = start[e] = 0;
    const int64_t last = (blockIdx.x + 1) * a.per_block < a.portions ? (blockIdx.x + 1) * a.per_block : a.portions;
    for (int64_t portion = blockIdx.x * a.per_block; portion < last; ++portion) {
        const int64_t s = portion / a.per_sequence, sequence_end = (s + 1) * a.sequence;
        const int64_t begin = s * a.sequence + portion % a.per_sequence * a.chunk;
        const int64_t end = begin + a.chunk < sequence_end ? begin + a.chunk : sequence_end;
        float sum[VALUES];
#pragma unroll
        for (int i = 0; i < VALUES; ++i) sum[i] = 0.0f;
        if (threadIdx.x == 0) counted_tokens = 0;
        if (!GIVEN)
            for (int i = threadIdx.x; i < a.experts * WORDS; i += THREADS) bits[i] = 0;
        __syncthreads();
        for (int64_t base = begin; base < end; base += ROWS) {
            const int64_t token = base + slot;
            const bool taken = token < end && (!a.mask || a.mask[token]);
            float l[VALUES];
            uint32_t key[VALUES], best = 0;
            if (taken) {
                load_logits<LANES, VALUES>(a, token, lane, l);
#pragma unroll
                for (int i = 0; i < VALUES; ++i) {
                    key[i] = key_of(l[i]);
                    best = key[i] > best ? key[i] : best;
                }
            } else {
#pragma unroll
                for (int i = 0; i < VALUES; ++i) { l[i] = -__builtin_inff(); key[i] = 0; }
            }
            best = lanes_max<LANES>(best);
            const bool counted = best != 0;
            const float m = value_of(best);
            float u[VALUES], all = 0.0f;
#pragma unroll
            for (int i = 0; i < VALUES; ++i) {
                u[i] = counted ? score(a.sigmoid, l[i], m) : 0.0f;
                all += u[i];
            }
            all = lanes_sum<LANES>(all);
            const float inverse = counted ? 1.0f / all : 0.0f;
#pragma unroll
            for (int i = 0; i < VALUES; ++i)
                if (counted) sum[i] = fmaf(u[i], inverse, sum[i]);
            if (lane == 0 && token < end) {
                if (a.stats) a.stats[token] = make_float2(counted ? m : 0.0f, inverse);
                if (counted) atomicAdd(&counted_tokens, 1);
            }
            if constexpr (GIVEN) {
                if (counted)
                    for (int j = lane; j < a.top_k; j += LANES) {
                        const int64_t at = token * a.top_k + j;
                        const int64_t e = a.given_wide ? static_cast<const int64_t*>(a.given)[at] : static_cast<const int*>(a.given)[at];
                        if (e >= 0 && e < a.experts) atomicAdd(&counts[e], 1);
                    }
            } else {
                float picked = 0.0f;
                for (int j = 0; j < a.top_k; ++j) {
                    if (j) {
                        best = 0;
#pragma unroll
                        for (int i = 0; i < VALUES; ++i) best = key[i] > best ? key[i] : best;
                        best = lanes_max<LANES>(best);
                    }
                    uint32_t first = 0xffffffffu;
#pragma unroll
                    for (int i = VALUES - 1; i >= 0; --i)
                        if (key[i] == best) first = (uint32_t)expert_of<LANES>(i, lane);
                    first = lanes_min<LANES>(first);
#pragma unroll
                    for (int i = 0; i < VALUES; ++i)
                        if (first == (uint32_t)expert_of<LANES>(i, lane)) key[i] = 0;
                    const float v = value_of(best);
                    const float value = best == 0 ? 0.0f : !a.normalize && a.sigmoid ? sigmoid_of(v) : score(a.sigmoid, v, m);
                    picked += value;
                    if (lane == 0) {
                        chosen[slot * a.top_k + j] = best == 0 ? -1 : (int)first;
                        values[slot * a.top_k + j] = value;
                        if (best != 0) atomicOr(&bits[first * WORDS + slot / 32], 1u << (slot % 32));
                    }
                }
                if (lane == 0) factors[slot] = a.scale * (a.normalize ? (counted ? 1.0f / picked : 0.0f) : a.sigmoid ? 1.0f : inverse);
                __syncthreads();
                for (int i = threadIdx.x; i < ROWS * a.top_k; i += THREADS) {
                    const int r = i / a.top_k;
                    if (base + r >= end) break;
                    const int e = chosen[i];
                    const int64_t at = base * a.top_k + i;
                    int place = -1;
                    if (e >= 0) {
                        place = counts[e];
                        for (int w = 0; w < r / 32; ++w) place += __popc(bits[e * WORDS + w]);
                        place += __popc(bits[e * WORDS + r / 32] & ((1u << (r % 32)) - 1u));
                    }
                    a.chosen[at] = e;
                    a.positions[at] = place;                                 // within the block; `places` adds the rest
                    a.gates[at] = e >= 0 ? values[i] * factors[r] : 0.0f;
                }
                __syncthreads();
                for (int e = threadIdx.x; e < a.experts; e += THREADS) {
                    int more = 0;
#pragma unroll
                    for (int w = 0; w < WORDS; ++w) {
                        more += __popc(bits[e * WORDS + w]);
                        bits[e * WORDS + w] = 0;
                    }
                    counts[e] += more;
                }
                __syncthreads();
            }
        }
        __syncthreads();
        // the portion's probabilities: over the rows of a wavefront, then over the wavefronts
#pragma unroll
        for (int i = 0; i < VALUES; ++i) {
            float v = sum[i];
#pragma unroll
            for (int d = LANES; d < 64; d *= 2) v += __shfl_xor(v, d, WAVE);
            const int e = expert_of<LANES>(i, lane);
            if (threadIdx.x % 64 < LANES && e < a.experts) sums[threadIdx.x / 64 * a.experts + e] = v;
        }
        __syncthreads();
        for (int e = threadIdx.x; e < a.experts; e += THREADS) {
            float v = sums[e];
#pragma unroll
            for (int w = 1; w < THREADS / 64; ++w) v += sums[w * a.experts + e];
            a.portion_sums[portion * a.experts + e] = v;
            a.portion_counts[portion * a.experts + e] = counts[e] - start[e];
            start[e] = counts[e];
        }
        if (threadIdx.x == 0) a.portion_tokens[portion] = counted_tokens;
        __syncthreads();
    }
    if (a.per_block > 1)
        for (int e = threadIdx.x; e < a.experts; e += THREADS) a.block_counts[blockIdx.x * a.experts + e] = counts[e];
    if (a.blocks > 1) return;
    // the only block: the rest of the work too
    __syncthreads();
    int *total = lds, *base = lds + a.experts;
    places(a, 0, total, base);
    if (!GIVEN)
        for (int64_t i = threadIdx.x; i < a.tokens * a.top_k; i += THREADS)
            if (a.chosen[i] >= 0) a.positions[i] += base[a.chosen[i]];
    __syncthreads();
    balance(a, reinterpret_cast<float*>(rest), rest + 2 * THREADS, slots);
}

// Blocks 0 .. blocks - 1: the places of each block's choices (choices made elsewhere have none: block 0 only, for the counts). The last
// block: the loss.
__global__ __launch_bounds__(1024) void place_kernel(RouteArgs a) {
    __shared__ int total[MOST_EXPERTS], base[MOST_EXPERTS], tokens[MOST_BLOCKS];
    __shared__ float piece[2 * 1024];
    __shared__ float2 slots[2][16];
    if (blockIdx.x == gridDim.x - 1) {
        balance(a, piece, tokens, slots);
        return;
    }
    const int64_t block = blockIdx.x;
    places(a, block, total, base);
    if (!a.positions) return;
    const int64_t first = block * a.per_block, last = first + a.per_block < a.portions ? first + a.per_block : a.portions;
    auto start_of = [&](int64_t portion) {
        const int64_t s = portion / a.per_sequence, at = s * a.sequence + portion % a.per_sequence * a.chunk, end = (s + 1) * a.sequence;
        return at < end ? at : end;
    };
    const int64_t end = (last == a.portions ? a.tokens : start_of(last)) * a.top_k;
    for (int64_t i = start_of(first) * a.top_k + threadIdx.x; i < end; i += blockDim.x) {
        const int e = a.chosen[i];
        if (e >= 0) a.positions[i] += base[e];
    }
}

// ---------------------------------------------------------------------------------------------------- backward
struct RouteGradArgs {
    RouteArgs r;                                                             // logits, shapes, chosen, stats and cost
    const float *dgates, *dloss;                                             // null: no gradient
    void* dlogits;
};

template <int LANES, int VALUES> __global__ __launch_bounds__(256) void route_gradient_kernel(RouteGradArgs g) {
    const RouteArgs& a = g.r;
    const int lane = threadIdx.x % LANES;
    const float dloss = g.dloss ? *g.dloss : 0.0f;
    for (int64_t token = (int64_t)blockIdx.x * (256 / LANES) + threadIdx.x / LANES; token < a.tokens; token += (int64_t)gridDim.x * (256 / LANES)) {
        const float2 stat = a.stats[token];
        float d[VALUES];
#pragma unroll
        for (int i = 0; i < VALUES; ++i) d[i] = 0.0f;
        if (stat.y != 0.0f) {                                                // a counted token (NaN too)
            float l[VALUES], p[VALUES], pull[VALUES];
            load_logits<LANES, VALUES>(a, token, lane, l);
            const float* cost = a.cost + token / a.sequence * a.experts;
            float towards = 0.0f;
#pragma unroll
            for (int i = 0; i < VALUES; ++i) {
                const int e = expert_of<LANES>(i, lane);
                p[i] = score(a.sigmoid, l[i], stat.x) * stat.y;
                pull[i] = g.dloss && e < a.experts ? dloss * cost[e] : 0.0f;
                towards = fmaf(p[i], pull[i], towards);
            }
            if (g.dgates) {
                float part[VALUES], picked = 0.0f, along = 0.0f;             // dgate where chosen; sums of p and p dgate over the chosen
                uint32_t chosen = 0;
#pragma unroll
                for (int i = 0; i < VALUES; ++i) part[i] = 0.0f;
                for (int j = 0; j < a.top_k; ++j) {
                    const int e = a.chosen[token * a.top_k + j];
                    const float dg = a.scale * g.dgates[token * a.top_k + j];
#pragma unroll
                    for (int i = 0; i < VALUES; ++i)
                        if (e == expert_of<LANES>(i, lane)) {
                            chosen |= 1u << i;
                            part[i] = dg;
                            picked += p[i];
                            along = fmaf(p[i], dg, along);
                        }
                }
                picked = lanes_sum<LANES>(picked);
                along = lanes_sum<LANES>(along);
                if (a.normalize) {                                           // gate_i = scale p_i / picked; its part of `towards` is zero
                    const float inverse = 1.0f / picked, mean = along * inverse;
#pragma unroll
                    for (int i = 0; i < VALUES; ++i)
                        if (chosen & (1u << i)) pull[i] = fmaf(part[i] - mean, inverse, pull[i]);
                } else if (!a.sigmoid) {                                     // gate_i = scale p_i
#pragma unroll
                    for (int i = 0; i < VALUES; ++i) pull[i] += part[i];
                    towards += lane == 0 ? along : 0.0f;
                } else {                                                     // gate_i = scale sigmoid(l_i)
#pragma unroll
                    for (int i = 0; i < VALUES; ++i)
                        if (chosen & (1u << i)) d[i] = part[i] * sigmoid_of(l[i]);
                }
            }
            towards = lanes_sum<LANES>(towards);
#pragma unroll
            for (int i = 0; i < VALUES; ++i) {
                d[i] = fmaf(p[i], pull[i] - towards, d[i]);
                if (a.sigmoid) d[i] *= sigmoid_of(-l[i]);
            }
        }
#pragma unroll
        for (int i = 0; i < VALUES; ++i) {
            const int e = expert_of<LANES>(i, lane);
            if (e < a.experts) store_float(g.dlogits, token * a.experts + e, a.dtype, d[i]);
        }
    }
}

// ---------------------------------------------------------------------------------------------------- launches
// calls f(lanes, values): the fewest lanes whose logits fit
template <typename F> void with_shape(int experts, F&& f) {
    if (experts <= 8) f(std::integral_constant<int, 2>(), std::integral_constant<int, 4>());
    else if (experts <= 16) f(std::integral_constant<int, 4>(), std::integral_constant<int, 4>());
    else if (experts <= 32) f(std::integral_constant<int, 8>(), std::integral_constant<int, 4>());
    else if (experts <= 64) f(std::integral_constant<int, 16>(), std::integral_constant<int, 4>());
    else if (experts <= 128) f(std::integral_constant<int, 16>(), std::integral_constant<int, 8>());
    else if (experts <= 256) f(std::integral_constant<int, 16>(), std::integral_constant<int, 16>());
    else if (experts <= 512) f(std::integral_constant<int, 64>(), std::integral_constant<int, 8>());
    else f(std::integral_constant<int, 64>(), std::integral_constant<int, 16>());
}

int lanes_for(int64_t experts) { return experts <= 8 ? 2 : experts <= 16 ? 4 : experts <= 32 ? 8 : experts <= 256 ? 16 : 64; }

// How the tokens are cut: portions of one sequence each, and portions of a block.
void plan(RouteArgs& a) {
    const int64_t rows = THREADS / lanes_for(a.experts);                     // tokens that a block takes at once
    const int64_t most = (MOST_BLOCKS + a.sequences - 1) / a.sequences, needed = (a.sequence + rows - 1) / rows;
    const int64_t cuts = a.sequences >= MOST_BLOCKS ? 1 : most < needed ? most : needed;
    a.chunk = ((a.sequence + cuts - 1) / cuts + rows - 1) / rows * rows;
    a.per_sequence = (a.sequence + a.chunk - 1) / a.chunk;
    a.portions = a.sequences * a.per_sequence;
    a.per_block = (a.portions + MOST_BLOCKS - 1) / MOST_BLOCKS;
    a.blocks = (a.portions + a.per_block - 1) / a.per_block;
}

int set_common(RouteArgs& a, const void* logits, int64_t pitch, int dtype, int64_t tokens, int64_t experts, int top_k, int score, int normalize, float scale,
               const uint8_t* mask, int64_t sequence) {
    VIOLA_CHECK_ARG(viola_is_float(dtype) && tokens >= 0 && experts > 0 && top_k > 0 && sequence > 0 && tokens % sequence == 0);
    VIOLA_CHECK_ARG((score == VIOLA_SOFTMAX || score == VIOLA_SIGMOID) && pitch >= experts);
    if (experts > MOST_EXPERTS || top_k > MOST_CHOSEN) return VIOLA_EUNSUPPORTED;
    VIOLA_CHECK_ARG(tokens < (1LL << 31) / MOST_CHOSEN);
    const size_t unit = dtype == VIOLA_F32 ? 16 : 8;
    a.logits = logits; a.pitch = pitch; a.dtype = dtype; a.tokens = tokens; a.experts = (int)experts; a.top_k = top_k;
    a.sigmoid = score == VIOLA_SIGMOID; a.normalize = normalize; a.scale = scale; a.mask = mask;
    a.whole = experts % 4 == 0 && pitch % 4 == 0 && reinterpret_cast<uintptr_t>(logits) % unit == 0;
    a.sequence = sequence; a.sequences = tokens / sequence;
    return 0;
}

// floats: sums of the portions; integers: counts of the portions and of the blocks, tokens of the portions
int64_t workspace_words(const RouteArgs& a) {
    return a.portions * a.experts * 2 + (a.per_block > 1 ? a.blocks * a.experts : 0) + a.portions;
}

int forward(RouteArgs& a, int32_t* workspace, int64_t words, hipStream_t stream) {
    plan(a);
    VIOLA_CHECK_ARG(workspace && words >= workspace_words(a));
    a.portion_sums = reinterpret_cast<float*>(workspace);
    a.portion_counts = workspace + a.portions * a.experts;
    a.portion_tokens = a.portion_counts + a.portions * a.experts;
    a.block_counts = a.per_block > 1 ? a.portion_tokens + a.portions : a.portion_counts;
    with_shape(a.experts, [&](auto lanes, auto values) {
        constexpr int LANES = decltype(lanes)::value, VALUES = decltype(values)::value;
        const unsigned lds = (unsigned)choose_lds<LANES>(a.experts, a.top_k, a.given != nullptr);
        if (a.given) VIOLA_LAUNCH((choose_kernel<LANES, VALUES, true>), dim3((unsigned)a.blocks), THREADS, lds, stream, a);
        else VIOLA_LAUNCH((choose_kernel<LANES, VALUES, false>), dim3((unsigned)a.blocks), THREADS, lds, stream, a);
    });
    if (a.blocks > 1) VIOLA_LAUNCH(place_kernel, dim3(a.given ? 2 : (unsigned)a.blocks + 1), 1024, 0, stream, a);
    return viola_launch_status();
}

}  // namespace

extern "C" int64_t viola_route_workspace(int64_t tokens, int64_t experts, int64_t sequence) {
    if (tokens <= 0 || experts <= 0 || experts > MOST_EXPERTS || sequence <= 0 || tokens % sequence) return 0;
    RouteArgs a = {};
    a.tokens = tokens; a.experts = (int)experts; a.sequence = sequence; a.sequences = tokens / sequence;
    plan(a);
    return workspace_words(a);
}

extern "C" int viola_route_forward(const void* logits, int64_t pitch, int dtype, int64_t tokens, int64_t experts, int top_k, int score, int normalize, float scale,
                                   const uint8_t* mask, int64_t sequence, int32_t* chosen, float* gates, int32_t* positions, int32_t* counts, int32_t* offsets,
                                   float* loss, float* cost, float* stats, int32_t* workspace, int64_t workspace_words, viola_stream_t stream_) {
    hipStream_t stream = viola_enter(stream_);
    RouteArgs a = {};
    if (const int status = set_common(a, logits, pitch, dtype, tokens, experts, top_k, score, normalize, scale, mask, sequence)) return status;
    VIOLA_CHECK_ARG(top_k <= experts);
    if (tokens == 0) return 0;
    VIOLA_CHECK_ARG(logits && chosen && gates && positions && counts && offsets && loss && cost && reinterpret_cast<uintptr_t>(stats) % 8 == 0);
    a.chosen = chosen; a.gates = gates; a.positions = positions; a.counts = counts; a.offsets = offsets; a.loss = loss; a.cost = cost;
    a.stats = reinterpret_cast<float2*>(stats);
    return forward(a, workspace, workspace_words, stream);
}

extern "C" int viola_balance_forward(const void* logits, int64_t pitch, int dtype, int64_t tokens, int64_t experts, int top_k, int score, const uint8_t* mask,
                                     int64_t sequence, const void* chosen, int chosen_wide, int32_t* counts, float* loss, float* cost, float* stats, int32_t* workspace,
                                     int64_t workspace_words, viola_stream_t stream_) {
    hipStream_t stream = viola_enter(stream_);
    RouteArgs a = {};
    if (const int status = set_common(a, logits, pitch, dtype, tokens, experts, top_k, score, 0, 1.0f, mask, sequence)) return status;
    if (tokens == 0) return 0;
    VIOLA_CHECK_ARG(logits && chosen && counts && loss && cost && reinterpret_cast<uintptr_t>(stats) % 8 == 0);
    a.given = chosen; a.given_wide = chosen_wide; a.counts = counts; a.loss = loss; a.cost = cost;
    a.stats = reinterpret_cast<float2*>(stats);
    return forward(a, workspace, workspace_words, stream);
}

extern "C" int viola_route_backward(const void* logits, int64_t pitch, int dtype, int64_t tokens, int64_t experts, int top_k, int score, int normalize, float scale,
                                    int64_t sequence, const int32_t* chosen, const float* cost, const float* stats, const float* dgates, const float* dloss,
                                    void* dlogits, viola_stream_t stream_) {
    hipStream_t stream = viola_enter(stream_);
    RouteGradArgs g = {};
    if (const int status = set_common(g.r, logits, pitch, dtype, tokens, experts, top_k, score, normalize, scale, nullptr, sequence)) return status;
    if (tokens == 0) return 0;
    VIOLA_CHECK_ARG(logits && dlogits && stats && (!dgates || chosen) && (!dloss || cost) && reinterpret_cast<uintptr_t>(stats) % 8 == 0);
    g.r.chosen = const_cast<int32_t*>(chosen);
    g.r.cost = const_cast<float*>(cost);
    g.r.stats = reinterpret_cast<float2*>(const_cast<float*>(stats));
    g.dgates = dgates; g.dloss = dloss; g.dlogits = dlogits;
    with_shape(g.r.experts, [&](auto lanes, auto values) {
        constexpr int LANES = decltype(lanes)::value, VALUES = decltype(values)::value;
        const int64_t blocks = (tokens + 256 / LANES - 1) / (256 / LANES);
        VIOLA_LAUNCH((route_gradient_kernel<LANES, VALUES>), dim3((unsigned)(blocks < 8192 ? blocks : 8192)), 256, 0, stream, g);
    });
    return viola_launch_status();
}
