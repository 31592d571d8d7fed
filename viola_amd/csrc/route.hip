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
// each token in LDS, blocks leave their counts and sums behind, and a second kernel adds those of the blocks before. Tokens of one stage (128;
// 256 of up to 16 experts, 512 of up to 8) in one sequence are one block's, which finishes by itself.
//
// Bound by instructions, not by memory: a wavefront spends some 860 of them on four rows of 128 logits, 55 on each choice (largest, its lowest index, taking it
// out), and the vector units are busy 70 % of the time. 32768 tokens to eight of 128 experts: choosing 18 us (its logits and results are 4 us of traffic), places and
// loss 9, gradient 11; two of 16 experts chosen elsewhere, 16384 tokens: 6, 5 and 3.4. Measured and left out, as neither was faster: a lane's logits sorted
// first (rank and expert as one double), a lane's largest found together with its index. 32 tokens, one block: 8.6 us, of which 4 are any
// launch, 1.6 the eight choices.
#include "block_ops.hpp"

#include <type_traits>

using namespace viola;

namespace {

constexpr int STAGE = 128, PLACE_THREADS = 512, MOST_EXPERTS = 1024, MOST_CHOSEN = 32, MOST_BLOCKS = 256;
constexpr int64_t MOST_TOKENS = (int64_t{1} << 31) / MOST_CHOSEN;            // so that choices are counted in 32 bits

struct RouteArgs {
    const void* logits;
    int64_t pitch, tokens;
    int dtype, experts, top_k, sigmoid, normalize, whole;                    // whole: rows can be read four logits at a time
    float scale;
    const uint8_t* mask;
    int64_t sequence, sequences, per_sequence, chunk, portions, per_block, blocks;
    int threads;                                                             // of a block that chooses
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
    if constexpr (LANES >= 32) {                                             // of a value and itself: rows 0 0 2 2 and rows 1 1 3 3 of 16 lanes
        const auto pair = __builtin_amdgcn_permlane16_swap(v, v, false, false);
        v = f(pair[0], pair[1]);
    }
    if constexpr (LANES >= 64) {                                             // the lower half twice and the upper half twice
        const auto pair = __builtin_amdgcn_permlane32_swap(v, v, false, false);
        v = f(pair[0], pair[1]);
    }
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

// exp(x) for x <= 0, within 2 ulp where that is a normal number, x >= -87.3: exp2 of the product's two halves, the low one multiplied in afterwards. What is smaller
// than 2^-126 comes out as 0, as the hardware's exp2 has no subnormal results; the last line is for -inf, whose halves are no numbers.
__device__ __forceinline__ float exp_of(float x) {
    const float t = x * 1.44269502f;                                         // log2(e) = 1.44269502 + 1.92596e-8
    const float low = fmaf(x, 1.92596299e-8f, fmaf(x, 1.44269502f, -t));
    const float e = __builtin_amdgcn_exp2f(t) * fmaf(low, 0.693147182f, 1.0f);
    return x < -150.0f ? 0.0f : e;
}

// u of a logit in a row whose largest is m
template <bool SIGMOID> __device__ __forceinline__ float score(float l, float m) {
    if constexpr (!SIGMOID) return exp_of(l - m);
    const float t = exp_of(-fabsf(l));                                       // sigmoid(l) = exp(min(l, 0)) / (1 + exp(-|l|))
    return exp_of(fminf(l, 0.0f) - fminf(m, 0.0f)) / (1.0f + t);
}
__device__ __forceinline__ float sigmoid_of(float l) {
    const float t = exp_of(-fabsf(l));
    return (l < 0.0f ? t : 1.0f) / (1.0f + t);
}

// VALUES logits of a lane: runs of four, LANES runs apart; -inf beyond the experts
template <int LANES> __device__ __forceinline__ int expert_of(int i, int lane) { return ((i / 4) * LANES + lane) * 4 + i % 4; }

template <int LANES, int VALUES, typename T> __device__ __forceinline__ void load_logits_as(const RouteArgs& a, int64_t token, int lane, float (&l)[VALUES]) {
    const T* row = static_cast<const T*>(a.logits) + token * a.pitch;
#pragma unroll
    for (int i = 0; i < VALUES; ++i) l[i] = -__builtin_inff();
    if (a.whole) {                                                           // experts is a multiple of four
#pragma unroll
        for (int i = 0; i < VALUES; i += 4) {
            const int e = expert_of<LANES>(i, lane);
            if (e >= a.experts) continue;
            if constexpr (sizeof(T) == 4) {
                const float4 v = *reinterpret_cast<const float4*>(row + e);
                l[i] = v.x; l[i + 1] = v.y; l[i + 2] = v.z; l[i + 3] = v.w;
            } else {
                const uint2 v = *reinterpret_cast<const uint2*>(row + e);
                l[i] = widen16<T>(v.x & 0xffffu); l[i + 1] = widen16<T>(v.x >> 16);
                l[i + 2] = widen16<T>(v.y & 0xffffu); l[i + 3] = widen16<T>(v.y >> 16);
            }
        }
    } else {
#pragma unroll
        for (int i = 0; i < VALUES; ++i)
            if (expert_of<LANES>(i, lane) < a.experts) l[i] = to_f32<T>(row[expert_of<LANES>(i, lane)]);
    }
}
template <int LANES, int VALUES> __device__ __forceinline__ void load_logits(const RouteArgs& a, int64_t token, int lane, float (&l)[VALUES]) {
    if (a.dtype == VIOLA_F32) load_logits_as<LANES, VALUES, float>(a, token, lane, l);
    else if (a.dtype == VIOLA_BF16) load_logits_as<LANES, VALUES, bf16_t>(a, token, lane, l);
    else load_logits_as<LANES, VALUES, f16_t>(a, token, lane, l);
}

// ---------------------------------------------------------------------------------------------------- after the blocks
// What a block leaves behind lies in rows of whole quads of experts, so that few wide loads are enough to add the rows of many blocks.
__host__ __device__ __forceinline__ int quads_of(int experts) { return (experts + 3) / 4; }
__device__ __forceinline__ int power_above(int n) {
    int wide = 1;
    while (wide < n) wide *= 2;
    return wide;
}

// Exclusive sums of total over the experts added to base (one wavefront: each lane a run of experts, then over the lanes); where
// `results`, counts and offsets go out.
__device__ __forceinline__ void add_offsets(const RouteArgs& a, const int* total, int* base, bool results) {
    if (threadIdx.x >= 64) return;
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
        if (results) {
            a.counts[e] = total[e];
            if (a.offsets) a.offsets[e] = at;
        }
        at += total[e];
    }
    if (results && a.offsets && threadIdx.x == 63) a.offsets[a.experts] = inclusive;
}

// Sums over the slices of a block's threads, of which thread t has column t % wide (a power of two) of slice t / wide: over the lanes of
// a wavefront, then over what is left in LDS ([blockDim] each), in one order. In threads below wide.
template <int N, typename T> __device__ __forceinline__ void over_slices(T (&v)[N], int wide, T (*lds)[PLACE_THREADS]) {
    for (int d = wide; d < 64; d *= 2) {
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] += __shfl_xor(v[i], d, WAVE);
    }
    const int lane = threadIdx.x % 64, parts = wide < 64 ? (int)blockDim.x / 64 : (int)blockDim.x / wide;
    if (wide >= 64 || lane < wide) {
#pragma unroll
        for (int i = 0; i < N; ++i) lds[i][wide >= 64 ? threadIdx.x : threadIdx.x / 64 * wide + lane] = v[i];
    }
    __syncthreads();
    if ((int)threadIdx.x < wide) {
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = lds[i][threadIdx.x];
#pragma unroll 4
        for (int u = 1; u < parts; ++u) {
#pragma unroll
            for (int i = 0; i < N; ++i) v[i] += lds[i][u * wide + threadIdx.x];
        }
    }
    __syncthreads();
}

// base[e]: the place of the first choice of e in `block`. Every thread of the block has to call it; total, base: [4 quads] in LDS.
__device__ __forceinline__ void places(const RouteArgs& a, int64_t block, int* total, int* base, int (*lds)[PLACE_THREADS]) {
    const int quads = quads_of(a.experts), wide = power_above(quads), slices = (int)blockDim.x / wide;      // 256 quads at most
    const int q = threadIdx.x % wide;
    int sum[8] = {};                                                         // of all blocks, and of those before
    if (q < quads) {
#pragma unroll 8
        for (int b = threadIdx.x / wide; b < (int)a.blocks; b += slices) {
            const int4 c = reinterpret_cast<const int4*>(a.block_counts)[b * quads + q];
            const int is = b < block;
            sum[0] += c.x; sum[1] += c.y; sum[2] += c.z; sum[3] += c.w;
            sum[4] += is * c.x; sum[5] += is * c.y; sum[6] += is * c.z; sum[7] += is * c.w;
        }
    }
    over_slices(sum, wide, lds);
    if ((int)threadIdx.x < quads) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            total[4 * q + i] = sum[i];
            base[4 * q + i] = sum[4 + i];
        }
    }
    __syncthreads();
    add_offsets(a, total, base, block == 0);
    __syncthreads();
}

// E c / (n^2 k sequences): how much the loss grows with a token's probability of e
__device__ __forceinline__ float cost_of(const RouteArgs& a, int count, int tokens) {
    const float n = (float)tokens;
    return tokens > 0 ? (float)a.experts * (float)count / (n * n * (float)a.top_k * (float)a.sequences) : 0.0f;
}

// The loss and the experts' costs, by one block: units (sequence, quad of experts), each of the portions of its sequence.
__device__ __forceinline__ void balance(const RouteArgs& a, float (*lds)[PLACE_THREADS], float2 (*slots)[16]) {
    const int m = (int)a.per_sequence, quads = quads_of(a.experts);
    const int64_t units = a.sequences * quads;
    const int wide = units < (int64_t)blockDim.x ? power_above((int)units) : (int)blockDim.x;
    const int slices = (int)blockDim.x / wide, slice = (int)threadIdx.x / wide;
    float loss = 0.0f;
    for (int64_t first = 0; first < units; first += wide) {
        const int64_t unit = first + threadIdx.x % wide, s = unit / quads;
        const int q = (int)(unit % quads);
        float sum[4] = {};
        int count[5] = {};                                                   // and tokens
        if (unit < units) {
#pragma unroll 8
            for (int64_t p = s * m + slice; p < (s + 1) * m; p += slices) {
                const float4 v = reinterpret_cast<const float4*>(a.portion_sums)[p * quads + q];
                const int4 c = reinterpret_cast<const int4*>(a.portion_counts)[p * quads + q];
                sum[0] += v.x; sum[1] += v.y; sum[2] += v.z; sum[3] += v.w;
                count[0] += c.x; count[1] += c.y; count[2] += c.z; count[3] += c.w;
                count[4] += a.portion_tokens[p];
            }
        }
        if (slices > 1) {                                                    // the units fit the block: one turn of this loop
            over_slices(sum, wide, lds);
            over_slices(count, wide, reinterpret_cast<int (*)[PLACE_THREADS]>(lds));
        }
        if (unit < units && slice == 0) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if (4 * q + i >= a.experts) break;
                const float cost = cost_of(a, count[i], count[4]);
                a.cost[s * a.experts + 4 * q + i] = cost;
                loss = fmaf(cost, sum[i], loss);
            }
        }
    }
    loss = BlockSums(slots).one(loss);
    if (threadIdx.x == 0) *a.loss = loss;
}

// ---------------------------------------------------------------------------------------------------- forward
// A block takes its tokens in stages: wavefronts choose for the rows of a stage each for itself, leaving the choices and a bit for each (expert, row)
// in LDS; then the places of all the stage's choices are read off the bits together.
// Four logits a lane up to 64 experts, eight to 512, sixteen beyond: one to four loads of up to 16 bytes and one to six steps over lanes.
// LDS: running counts and counts at the portion's start [4 quads] each, bits [experts][words], chosen and values [stage * top_k], factors
// [stage], then sums [8][experts] (over the bits and what follows them, once a portion is done)
// Threads of a block at most: four wavefronts for a SIMD where their registers fit, as choosing is a chain of short dependent steps (32768 tokens to eight of
// 128: 18.2 us; with 512 threads at most 19.8, with 256 29.3).
template <int VALUES> __host__ __device__ constexpr int threads_of() { return VALUES <= 8 ? 1024 : 512; }
// Tokens of a stage: as many as that at once, STAGE at least
template <int LANES, int VALUES> __host__ __device__ constexpr int stage_of() { return threads_of<VALUES>() / LANES > STAGE ? threads_of<VALUES>() / LANES : STAGE; }

template <int LANES, int VALUES> size_t choose_lds(int experts, int top_k, bool given) {
    const size_t rows = stage_of<LANES, VALUES>();
    const size_t choice = given ? 0 : (size_t)experts * (rows / 32) + 2 * rows * top_k + rows;
    const size_t sums = (size_t)(threads_of<VALUES>() / 64) * experts;
    return 4 * (8 * (size_t)quads_of(experts) + (choice > sums ? choice : sums));
}

template <int LANES, int VALUES, bool GIVEN, bool SIGMOID> __global__ __launch_bounds__(threads_of<VALUES>()) void choose_kernel(RouteArgs a) {
    extern __shared__ int lds[];
    __shared__ int counted_tokens;
    __shared__ float2 slots[2][16];
    constexpr int STAGED = stage_of<LANES, VALUES>(), WORDS = STAGED / 32;
    const int threads = blockDim.x, rows = threads / LANES;
    const int quads = quads_of(a.experts);
    int *counts = lds, *start = lds + 4 * quads, *rest = lds + 8 * quads;
    uint32_t* bits = reinterpret_cast<uint32_t*>(rest);
    int* chosen = rest + a.experts * WORDS;
    float* values = reinterpret_cast<float*>(chosen + STAGED * a.top_k);
    float* factors = values + STAGED * a.top_k;
    float* sums = reinterpret_cast<float*>(rest);
    const int lane = threadIdx.x % LANES, slot = threadIdx.x / LANES;
    const bool alone = a.blocks == 1;                                        // then there is one portion of one stage, and nothing to leave behind
    for (int e = threadIdx.x; e < 4 * quads; e += threads) counts[e] = start[e] = 0;
    const int64_t last = (blockIdx.x + 1) * a.per_block < a.portions ? (blockIdx.x + 1) * a.per_block : a.portions;
    for (int64_t portion = blockIdx.x * a.per_block; portion < last; ++portion) {
        const int64_t s = portion / a.per_sequence, sequence_end = (s + 1) * a.sequence;
        const int64_t begin = s * a.sequence + portion % a.per_sequence * a.chunk;
        const int64_t end = begin + a.chunk < sequence_end ? begin + a.chunk : sequence_end;
        float sum[VALUES];
#pragma unroll
        for (int i = 0; i < VALUES; ++i) sum[i] = 0.0f;
        int here = 0;                                                        // tokens that the wavefront has counted
        float next[VALUES];
        bool next_taken;
        auto load = [&](int64_t token) {
            next_taken = token < end && (!a.mask || a.mask[token]);
            if (next_taken) {
                load_logits<LANES, VALUES>(a, token, lane, next);
            } else {
#pragma unroll
                for (int i = 0; i < VALUES; ++i) next[i] = -__builtin_inff();
            }
        };
        load(begin + slot);
        if (threadIdx.x == 0) counted_tokens = 0;
        if (!GIVEN)
            for (int i = threadIdx.x; i < a.experts * WORDS; i += threads) bits[i] = 0;
        __syncthreads();
        for (int64_t base = begin; base < end; base += STAGED) {
            for (int row = slot; row - slot < STAGED && base + row - slot < end; row += rows) {
                const int64_t token = base + row;
                float l[VALUES];
                uint32_t key[VALUES], best = 0;
#pragma unroll
                for (int i = 0; i < VALUES; ++i) {
                    l[i] = next[i];
                    key[i] = key_of(l[i]);                                   // 0 for a token that is left out
                    best = key[i] > best ? key[i] : best;
                }
                load(token + rows);
                best = lanes_max<LANES>(best);
                const bool counted = best != 0;
                const float m = value_of(best);
                float u[VALUES], all = 0.0f;
#pragma unroll
                for (int i = 0; i < VALUES; ++i) {
                    u[i] = score<SIGMOID>(l[i], m);
                    u[i] = counted ? u[i] : 0.0f;
                    all += u[i];
                }
                all = lanes_sum<LANES>(all);
                const float inverse = counted ? 1.0f / all : 0.0f;
#pragma unroll
                for (int i = 0; i < VALUES; ++i) sum[i] = fmaf(u[i], inverse, sum[i]);
                if (lane == 0 && token < end) {
                    if (a.stats) a.stats[token] = make_float2(counted ? m : 0.0f, inverse);
                }
                here += __popcll(__ballot(lane == 0 && counted));
                if constexpr (GIVEN) {
                    if (counted)
                        for (int j = lane; j < a.top_k; j += LANES) {
                            const int64_t at = token * a.top_k + j;
                            const int64_t e = a.given_wide ? static_cast<const int64_t*>(a.given)[at] : static_cast<const int*>(a.given)[at];
                            if (e >= 0 && e < a.experts) atomicAdd(&counts[e], 1);
                        }
                } else {
                    // LANES choices at a time, one left with each lane: its score and its bit are that lane's work
                    float picked = 0.0f;
                    for (int j0 = 0; j0 < a.top_k; j0 += LANES) {
                        const int more = a.top_k - j0 < LANES ? a.top_k - j0 : LANES;
                        uint32_t my_key = 0, my_expert = 0;
                        for (int j = 0; j < more; ++j) {
                            if (j0 + j) {
                                best = 0;
#pragma unroll
                                for (int i = 0; i < VALUES; ++i) best = key[i] > best ? key[i] : best;
                                best = lanes_max<LANES>(best);
                            }
                            uint32_t first = 0xffffffffu;
#pragma unroll
                            for (int i = VALUES - 1; i >= 0; --i) first = key[i] == best ? (uint32_t)expert_of<LANES>(i, lane) : first;
                            first = lanes_min<LANES>(first);
#pragma unroll
                            for (int i = 0; i < VALUES; ++i) key[i] = first == (uint32_t)expert_of<LANES>(i, lane) ? 0 : key[i];
                            my_key = lane == j ? best : my_key;
                            my_expert = lane == j ? first : my_expert;
                        }
                        if (lane < more) {
                            const float v = value_of(my_key);
                            const float value = !a.normalize && SIGMOID ? sigmoid_of(v) : score<SIGMOID>(v, m);
                            const int at = row * a.top_k + j0 + lane;
                            chosen[at] = my_key ? (int)my_expert : -1;
                            values[at] = value;
                            if (my_key) {
                                picked += value;
                                atomicOr(&bits[my_expert * WORDS + row / 32], 1u << (row % 32));
                            }
                        }
                    }
                    picked = lanes_sum<LANES>(picked);
                    if (lane == 0) factors[row] = a.scale * (a.normalize ? (counted ? 1.0f / picked : 0.0f) : SIGMOID ? 1.0f : inverse);
                }
            }
            if constexpr (!GIVEN) {
                __syncthreads();
                if (alone) {                                                 // start: the places' beginnings, at once
                    for (int e = threadIdx.x; e < a.experts; e += threads) {
                        int total = 0;
#pragma unroll
                        for (int w = 0; w < WORDS; ++w) total += __popc(bits[e * WORDS + w]);
                        counts[e] = total;
                    }
                    __syncthreads();
                    add_offsets(a, counts, start, true);
                    __syncthreads();
                }
                const int* from = alone ? start : counts;
                const int choices = (int)(end - base < STAGED ? end - base : STAGED) * a.top_k;
                for (int i = threadIdx.x; i < choices; i += threads) {
                    const int r = i / a.top_k, e = chosen[i];
                    const int64_t at = base * a.top_k + i;
                    int place = -1;
                    if (e >= 0) {
                        place = from[e] + __popc(bits[e * WORDS + r / 32] & ((1u << (r % 32)) - 1u));
                        for (int w = 0; w < r / 32; ++w) place += __popc(bits[e * WORDS + w]);
                    }
                    a.chosen[at] = e;
                    a.positions[at] = place;                                 // of several blocks, within this one: place_kernel adds the rest
                    a.gates[at] = e >= 0 ? values[i] * factors[r] : 0.0f;
                }
                __syncthreads();
                if (!alone) {
                    for (int e = threadIdx.x; e < a.experts; e += threads) {
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
        }
        if (threadIdx.x % 64 == 0) atomicAdd(&counted_tokens, here);
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
        float loss = 0.0f;
        for (int e = threadIdx.x; e < a.experts; e += threads) {
            float v = sums[e];
            for (int w = 1; w < threads / 64; ++w) v += sums[w * a.experts + e];
            if (alone) {
                const float cost = cost_of(a, counts[e], counted_tokens);
                a.cost[e] = cost;
                if (GIVEN) a.counts[e] = counts[e];
                loss = fmaf(cost, v, loss);
            } else {
                a.portion_sums[portion * 4 * quads + e] = v;
                a.portion_counts[portion * 4 * quads + e] = counts[e] - start[e];
                start[e] = counts[e];
            }
        }
        if (alone) {
            BlockSums block(slots);
            loss = block.one(loss);
            if (threadIdx.x == 0) *a.loss = loss;
            return;
        }
        if (threadIdx.x == 0) a.portion_tokens[portion] = counted_tokens;
        __syncthreads();
    }
    if (a.per_block > 1)
        for (int e = threadIdx.x; e < a.experts; e += threads) a.block_counts[blockIdx.x * 4 * quads + e] = counts[e];
}

// Block 0: the loss. Blocks 1 to `blocks`: the places of each block's choices (choices made elsewhere have none: one block only, for the
// counts). 512 threads, so that two blocks fit a CU: the loss takes longest and would otherwise have one more round to itself.
__global__ __launch_bounds__(PLACE_THREADS) void place_kernel(RouteArgs a) {
    __shared__ int total[MOST_EXPERTS], base[MOST_EXPERTS], pieces[8][PLACE_THREADS];
    __shared__ float2 slots[2][16];
    if (blockIdx.x == 0) {
        balance(a, reinterpret_cast<float (*)[PLACE_THREADS]>(pieces), slots);
        return;
    }
    const int64_t block = blockIdx.x - 1;
    const int64_t first = block * a.per_block, last = first + a.per_block < a.portions ? first + a.per_block : a.portions;
    auto start_of = [&](int64_t portion) {
        const int64_t s = portion / a.per_sequence, at = s * a.sequence + portion % a.per_sequence * a.chunk, end = (s + 1) * a.sequence;
        return at < end ? at : end;
    };
    const int64_t end = (last == a.portions ? a.tokens : start_of(last)) * a.top_k;
    int64_t i = start_of(first) * a.top_k + threadIdx.x;
    int e = -1, place = 0;                                                   // the first choice's loads are under way while the blocks are added
    if (a.positions && i < end) {
        e = a.chosen[i];
        place = a.positions[i];
    }
    places(a, block, total, base, pieces);
    while (a.positions && i < end) {
        if (e >= 0) a.positions[i] = place + base[e];
        i += blockDim.x;
        if (i >= end) break;
        e = a.chosen[i];
        place = a.positions[i];
    }
}

// ---------------------------------------------------------------------------------------------------- backward
struct RouteGradArgs {
    RouteArgs r;                                                             // logits, shapes, chosen, stats and cost
    const float *dgates, *dloss;                                             // null: no gradient
    void* dlogits;
    int whole;                                                               // its rows can be written four at a time
};

// What stands for "not chosen" among the gates' gradients in LDS: a NaN that none of them is, as theirs are made the usual one.
constexpr uint32_t NOT_CHOSEN = 0xffffdeadu;

template <int LANES, int VALUES, bool SIGMOID> __global__ __launch_bounds__(256) void route_gradient_kernel(RouteGradArgs g) {
    constexpr int ROWS = 256 / LANES;
    __shared__ uint32_t parts[ROWS][LANES * VALUES];                         // a row's gate gradients by expert; its own lanes' only
    const RouteArgs& a = g.r;
    const int lane = threadIdx.x % LANES, slot = threadIdx.x / LANES;
    const int tokens = (int)a.tokens, sequence = (int)a.sequence;            // below 2^26
    const float dloss = g.dloss ? *g.dloss : 0.0f;
    for (int first = blockIdx.x * ROWS; first < tokens; first += gridDim.x * ROWS) {
        const int token = first + slot;
        const bool there = token < tokens;
        float2 stat = make_float2(0.0f, 0.0f);
        float l[VALUES], pull[VALUES];
        uint32_t word[VALUES];                                               // scaled gradients of the gates, or NOT_CHOSEN
#pragma unroll
        for (int i = 0; i < VALUES; ++i) {
            l[i] = -__builtin_inff();
            pull[i] = 0.0f;
            word[i] = NOT_CHOSEN;
        }
        if (there) {
            stat = a.stats[token];
            load_logits<LANES, VALUES>(a, token, lane, l);
            if (g.dloss) {
                const float* cost = a.cost + (int64_t)(token / sequence) * a.experts;
                if (a.experts % 4 == 0) {
#pragma unroll
                    for (int i = 0; i < VALUES; i += 4)
                        if (expert_of<LANES>(i, lane) < a.experts) {
                            const float4 c = *reinterpret_cast<const float4*>(cost + expert_of<LANES>(i, lane));
                            pull[i] = dloss * c.x; pull[i + 1] = dloss * c.y; pull[i + 2] = dloss * c.z; pull[i + 3] = dloss * c.w;
                        }
                } else {
#pragma unroll
                    for (int i = 0; i < VALUES; ++i)
                        if (expert_of<LANES>(i, lane) < a.experts) pull[i] = dloss * cost[expert_of<LANES>(i, lane)];
                }
            }
        }
        const bool counted = stat.y != 0.0f;                                 // NaN is
        if (g.dgates) {
#pragma unroll
            for (int i = 0; i < VALUES; i += 4) *reinterpret_cast<uint4*>(&parts[slot][expert_of<LANES>(i, lane)]) = make_uint4(NOT_CHOSEN, NOT_CHOSEN, NOT_CHOSEN, NOT_CHOSEN);
            __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");           // a row's lanes are of one wavefront, whose LDS accesses stay in order
            __builtin_amdgcn_wave_barrier();
            if (there)
                for (int j = lane; j < a.top_k; j += LANES) {
                    const int e = a.chosen[(int64_t)token * a.top_k + j];
                    const float dg = a.scale * g.dgates[(int64_t)token * a.top_k + j];
                    if (e >= 0 && e < a.experts) parts[slot][e] = dg != dg ? 0x7fc00000u : __float_as_uint(dg);
                }
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            __builtin_amdgcn_wave_barrier();
#pragma unroll
            for (int i = 0; i < VALUES; i += 4) {
                const uint4 w = *reinterpret_cast<const uint4*>(&parts[slot][expert_of<LANES>(i, lane)]);
                word[i] = w.x; word[i + 1] = w.y; word[i + 2] = w.z; word[i + 3] = w.w;
            }
            __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
            __builtin_amdgcn_wave_barrier();
        }
        auto part = [&](int i) { return word[i] == NOT_CHOSEN ? 0.0f : __uint_as_float(word[i]); };
        float p[VALUES], from_gates[VALUES], towards = 0.0f, picked = 0.0f, along = 0.0f;    // sum of p pull; over the chosen, of p and of p dgate
#pragma unroll
        for (int i = 0; i < VALUES; ++i) {
            p[i] = score<SIGMOID>(l[i], stat.x) * stat.y;
            towards = fmaf(p[i], pull[i], towards);
            picked += word[i] == NOT_CHOSEN ? 0.0f : p[i];
            along = fmaf(p[i], part(i), along);
            from_gates[i] = 0.0f;
        }
        towards = lanes_sum<LANES>(towards);
        if (g.dgates && (a.normalize || !SIGMOID)) {
            if (a.normalize) {                                               // gate_i = scale q_i, q = p / picked: q_i (dgate_i - sum q dgate)
                picked = lanes_sum<LANES>(picked);
                const float inverse = 1.0f / picked;
                along = 0.0f;
#pragma unroll
                for (int i = 0; i < VALUES; ++i) {
                    // the quotient to its last place: of a row's only choice it is 1, whose gradient is 0 and not what rounding leaves of it
                    const float near = p[i] * inverse, q = fmaf(fmaf(-near, picked, p[i]), inverse, near);
                    from_gates[i] = word[i] == NOT_CHOSEN ? 0.0f : q;
                    along = fmaf(from_gates[i], part(i), along);
                }
                const float mean = lanes_sum<LANES>(along);
#pragma unroll
                for (int i = 0; i < VALUES; ++i) from_gates[i] = word[i] == NOT_CHOSEN ? 0.0f : from_gates[i] * (__uint_as_float(word[i]) - mean);
            } else {                                                         // gate_i = scale p_i
                along = lanes_sum<LANES>(along);
#pragma unroll
                for (int i = 0; i < VALUES; ++i) pull[i] += part(i);
                towards += along;
            }
        }
        float d[VALUES];
#pragma unroll
        for (int i = 0; i < VALUES; ++i) {
            d[i] = fmaf(p[i], pull[i] - towards, from_gates[i]);
            if constexpr (SIGMOID) {
                if (!a.normalize) d[i] = fmaf(part(i), sigmoid_of(l[i]), d[i]);                                // gate_i = scale sigmoid(l_i)
                d[i] *= sigmoid_of(-l[i]);
            }
            if (!counted) d[i] = 0.0f;
        }
        if (!there) continue;
#pragma unroll
        for (int i = 0; i < VALUES; i += 4) {
            const int e = expert_of<LANES>(i, lane);
            if (g.whole) {
                if (e >= a.experts) continue;
                const int64_t at = (int64_t)token * a.experts + e;
                if (a.dtype == VIOLA_F32) *reinterpret_cast<float4*>(static_cast<float*>(g.dlogits) + at) = make_float4(d[i], d[i + 1], d[i + 2], d[i + 3]);
                else if (a.dtype == VIOLA_BF16)
                    *reinterpret_cast<uint2*>(static_cast<uint16_t*>(g.dlogits) + at) = make_uint2(f32_to_bf16x2_bits(d[i], d[i + 1]), f32_to_bf16x2_bits(d[i + 2], d[i + 3]));
                else
                    *reinterpret_cast<uint2*>(static_cast<uint16_t*>(g.dlogits) + at) =
                        make_uint2(narrow16<f16_t>(d[i]) | narrow16<f16_t>(d[i + 1]) << 16, narrow16<f16_t>(d[i + 2]) | narrow16<f16_t>(d[i + 3]) << 16);
            } else {
#pragma unroll
                for (int c = 0; c < 4; ++c)
                    if (e + c < a.experts) store_float(g.dlogits, (int64_t)token * a.experts + e + c, a.dtype, d[i + c]);
            }
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
    else if (experts <= 256) f(std::integral_constant<int, 32>(), std::integral_constant<int, 8>());
    else if (experts <= 512) f(std::integral_constant<int, 64>(), std::integral_constant<int, 8>());
    else f(std::integral_constant<int, 64>(), std::integral_constant<int, 16>());
}

// How the tokens are cut: portions of one sequence each, and portions of a block.
void plan(RouteArgs& a) {
    int64_t rows = 0, staged = 0, lanes_of_row = 0;                          // tokens that a block takes at once, and in one stage
    with_shape(a.experts, [&](auto lanes, auto values) {
        lanes_of_row = decltype(lanes)::value;
        a.threads = threads_of<decltype(values)::value>();
        staged = stage_of<decltype(lanes)::value, decltype(values)::value>();
    });
    // half the threads where blocks of them are fewer than CUs; no more than a sequence's tokens have lanes, two wavefronts at least
    const int64_t used = (a.sequence * lanes_of_row + 127) / 128 * 128;
    if (a.threads == 1024 && a.tokens * lanes_of_row < 1024 * MOST_BLOCKS) a.threads = 512;
    if (used < a.threads) a.threads = (int)used;
    rows = a.threads / lanes_of_row;
    const int64_t most = (MOST_BLOCKS + a.sequences - 1) / a.sequences, needed = (a.sequence + rows - 1) / rows;
    const bool stage = a.sequences == 1 && a.tokens <= staged;                      // one block, one launch
    const int64_t cuts = stage || a.sequences >= MOST_BLOCKS ? 1 : most < needed ? most : needed;
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
    VIOLA_CHECK_ARG(tokens < MOST_TOKENS);
    const size_t unit = dtype == VIOLA_F32 ? 16 : 8;
    a.logits = logits; a.pitch = pitch; a.dtype = dtype; a.tokens = tokens; a.experts = (int)experts; a.top_k = top_k;
    a.sigmoid = score == VIOLA_SIGMOID; a.normalize = normalize; a.scale = scale; a.mask = mask;
    a.whole = experts % 4 == 0 && pitch % 4 == 0 && reinterpret_cast<uintptr_t>(logits) % unit == 0;
    a.sequence = sequence; a.sequences = tokens / sequence;
    return 0;
}

// sums and counts of the portions, counts of the blocks, tokens of the portions
int64_t workspace_words(const RouteArgs& a) {
    const int64_t row = 4 * quads_of(a.experts);
    return a.portions * row * 2 + (a.per_block > 1 ? a.blocks * row : 0) + a.portions;
}

int forward(RouteArgs& a, int32_t* workspace, int64_t words, hipStream_t stream) {
    plan(a);
    VIOLA_CHECK_ARG(workspace && words >= workspace_words(a) && reinterpret_cast<uintptr_t>(workspace) % 16 == 0);
    const int64_t row = 4 * quads_of(a.experts);
    a.portion_sums = reinterpret_cast<float*>(workspace);
    a.portion_counts = workspace + a.portions * row;
    a.block_counts = a.per_block > 1 ? a.portion_counts + a.portions * row : a.portion_counts;
    a.portion_tokens = a.portion_counts + (a.portions + (a.per_block > 1 ? a.blocks : 0)) * row;
    with_shape(a.experts, [&](auto lanes, auto values) {
        constexpr int LANES = decltype(lanes)::value, VALUES = decltype(values)::value;
        const unsigned lds = (unsigned)choose_lds<LANES, VALUES>(a.experts, a.top_k, a.given != nullptr);
        auto launch = [&](auto given, auto sigmoid) {
            VIOLA_LAUNCH((choose_kernel<LANES, VALUES, decltype(given)::value, decltype(sigmoid)::value>), dim3((unsigned)a.blocks), a.threads, lds, stream, a);
        };
        if (a.given) a.sigmoid ? launch(std::true_type(), std::true_type()) : launch(std::true_type(), std::false_type());
        else a.sigmoid ? launch(std::false_type(), std::true_type()) : launch(std::false_type(), std::false_type());
    });
    if (a.blocks > 1) VIOLA_LAUNCH(place_kernel, dim3(a.given ? 2 : (unsigned)a.blocks + 1), PLACE_THREADS, 0, stream, a);
    return viola_launch_status();
}

}  // namespace

extern "C" int64_t viola_route_workspace(int64_t tokens, int64_t experts, int64_t sequence) {
    if (tokens <= 0 || tokens >= MOST_TOKENS || experts <= 0 || experts > MOST_EXPERTS || sequence <= 0 || tokens % sequence) return 0;
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
    VIOLA_CHECK_ARG(logits && dlogits && stats && (!dgates || chosen) && (!dloss || cost) && reinterpret_cast<uintptr_t>(stats) % 8 == 0 &&
                    reinterpret_cast<uintptr_t>(cost) % 16 == 0);
    g.r.chosen = const_cast<int32_t*>(chosen);
    g.r.cost = const_cast<float*>(cost);
    g.r.stats = reinterpret_cast<float2*>(const_cast<float*>(stats));
    g.dgates = dgates; g.dloss = dloss; g.dlogits = dlogits;
    g.whole = experts % 4 == 0 && reinterpret_cast<uintptr_t>(dlogits) % 16 == 0;
    with_shape(g.r.experts, [&](auto lanes, auto values) {
        constexpr int LANES = decltype(lanes)::value, VALUES = decltype(values)::value;
        const int64_t blocks = (tokens + 256 / LANES - 1) / (256 / LANES);
        const dim3 grid((unsigned)(blocks < 8192 ? blocks : 8192));
        if (g.r.sigmoid) VIOLA_LAUNCH((route_gradient_kernel<LANES, VALUES, true>), grid, 256, 0, stream, g);
        else VIOLA_LAUNCH((route_gradient_kernel<LANES, VALUES, false>), grid, 256, 0, stream, g);
    });
    return viola_launch_status();
}
