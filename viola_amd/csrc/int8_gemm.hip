// Products of 8-bit integers with a scale for each row of either operand (tokens and channels), whole or by groups of rows.
//
// The integers are multiplied by v_mfma_i32_32x32x32_i8, whose 32-bit sums are exact; the scales are applied to the finished sums in registers:
// out = (sum * sa) * sb + bias, one rounding each. Bound by the matrix pipes (as many operations a cycle as FP8; why the first of these takes longer than the same tiles on FP8, 509 us,
// has not been found): 16384 x 4096 -> 11008 645 to 690 us (2.2 POP/s), 4096 x 11008 -> 4096 143 (2.6), 8192 x 1024 -> 4096 46 (1.5: the results of a round of tiles leave at its end, some 9 us of 23).
//
// The tiles are those of gemm_pingpong.hpp: eight wavefronts, two on each SIMD, whose memory work and math alternate; a chunk of 128 k is two pairs of
// instructions for each 32 x 32 sub-tile where FP8 has one of 64 k, and an operand's 16-byte pieces are in the instruction's own order.
#include <type_traits>

#include "gemm_pingpong.hpp"
#include "int8_args.hpp"
#include "int8_quantize.hpp"

namespace viola {

typedef int i32x16 __attribute__((ext_vector_type(16)));

typedef int loose_words4 __attribute__((ext_vector_type(4), aligned(2)));

// 16 bytes of a row from column `col` on, at any address: one store all the same
template <typename TO> __device__ __forceinline__ void store_piece(TO* to, int64_t col, int64_t n, const uint4& value) {
    constexpr int PER = 16 / (int)sizeof(TO);
    if (col + PER <= n) {
        __builtin_nontemporal_store(loose_words4{(int)value.x, (int)value.y, (int)value.z, (int)value.w}, reinterpret_cast<loose_words4*>(to));
    } else {
        const TO* values = reinterpret_cast<const TO*>(&value);
        for (int e = 0; e < PER; ++e)
            if (col + e < n) to[e] = values[e];
    }
}

// The finished sums of a wave times their scales plus bias, through its own part of the ring (which every wave has left), out in 16-byte pieces.
template <typename S, typename TO>
__device__ __forceinline__ void store_int8_tile(const i32x16 (&total)[S::TN][S::TM], const Int8Args& p, TO* out, int64_t m_begin, int64_t m_end, int64_t n_begin,
                                                uint8_t* ring, const float* columns) {
    const int lane = threadIdx.x % WAVE, l32 = lane % 32, lhi = lane / 32;
    const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x / WAVE), wm = wave / S::WN, wn = wave % S::WN;
    constexpr int PER = 16 / (int)sizeof(TO), COLS_W = 32 * S::TN, PLD = COLS_W + PER, PIECES = COLS_W / PER;
    static_assert(8 * 32 * PLD * (int)sizeof(TO) <= S::STAGES * S::STAGE);
    TO* park = reinterpret_cast<TO*>(ring) + wave * 32 * PLD;
    const int64_t ncol0 = n_begin + wn * COLS_W;
#pragma unroll
    for (int j = 0; j < S::TM; ++j) {
        const int64_t row0 = m_begin + (wm * S::TM + j) * 32;
        const RowFactor row(row0 + l32 < m_end ? p.sa[row0 + l32] : 0.0f);
#pragma unroll
        for (int i = 0; i < S::TN; ++i)
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const int col = (wn * S::TN + i) * 32 + q * 8 + lhi * 4;
                const float4 sb = *reinterpret_cast<const float4*>(&columns[col]), bias = *reinterpret_cast<const float4*>(&columns[S::COLS + col]);
                const float v[4] = {fmaf((float)total[i][j][4 * q] * row.s * sb.x, row.lift, bias.x), fmaf((float)total[i][j][4 * q + 1] * row.s * sb.y, row.lift, bias.y),
                                    fmaf((float)total[i][j][4 * q + 2] * row.s * sb.z, row.lift, bias.z), fmaf((float)total[i][j][4 * q + 3] * row.s * sb.w, row.lift, bias.w)};
                Quad<TO>::store(&park[l32 * PLD + i * 32 + q * 8 + lhi * 4], v);
            }
#pragma unroll
        for (int it = 0; it < 32 * PIECES / WAVE; ++it) {
            const int id = it * WAVE + lane, pr = id / PIECES, pc = id % PIECES;
            const int64_t mrow = row0 + pr, ncol = ncol0 + pc * PER;
            const uint4 value = *reinterpret_cast<const uint4*>(&park[pr * PLD + pc * PER]);
            if (mrow < m_end && ncol < p.n) store_piece(out + mrow * p.ldo + ncol, ncol, p.n, value);
        }
    }
}

// The same for the product dh of a gated activation's backward pass: dz = [dh u act'(g) | dh act(g)], dh in 32 bits from the wave's part of the ring, z read and dz written in
// pieces of eight columns along the rows. On pairs of blocks, one's activations under the other's products: 32768 rows at 64 experts, 1024 -> 1024, 102 to 125 us, as two passes 93 and 65,
// on tiles of 256 x 256, whose only block does nothing beside it, 158. Sums of more than GATED_MOST_K are two passes: there the larger tiles win more (.6 us for 64 k of
// 65536 results on a CU) than dh out and back in 32 bits costs.
template <typename S, typename TO>
__device__ __forceinline__ void store_int8_gradient(const i32x16 (&total)[S::TN][S::TM], const Int8Args& p, int64_t m_begin, int64_t m_end, int64_t n_begin, uint8_t* ring,
                                                    const float* columns) {
    const int lane = threadIdx.x % WAVE, l32 = lane % 32, lhi = lane / 32;
    const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x / WAVE), wm = wave / S::WN, wn = wave % S::WN;
    constexpr int COLS_W = 32 * S::TN, PLD = COLS_W + 4, PIECES = COLS_W / 8, TURNS = 32 * PIECES / WAVE;
    static_assert(8 * 32 * PLD * 4 <= S::STAGES * S::STAGE);
    float* park = reinterpret_cast<float*>(ring) + wave * 32 * PLD;
    const int64_t ncol0 = n_begin + wn * COLS_W;
#pragma unroll
    for (int j = 0; j < S::TM; ++j) {
        const int64_t row0 = m_begin + (wm * S::TM + j) * 32;
        Raw8<TO> g[TURNS], u[TURNS];
#pragma unroll
        for (int it = 0; it < TURNS; ++it) {
            const int id = it * WAVE + lane;
            const int64_t row = row0 + id / PIECES, col = ncol0 + id % PIECES * 8;
            const TO* z = static_cast<const TO*>(p.z) + row * p.z_pitch + col;
            const int left = (int)(p.n - col < 8 ? p.n - col : 8);
            if (row >= m_end || left <= 0) continue;
            g[it].load(z, 0, left);
            u[it].load(z + p.n, 0, left);
        }
        const float sa = row0 + l32 < m_end ? p.sa[row0 + l32] : 0.0f;
#pragma unroll
        for (int i = 0; i < S::TN; ++i)
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const float4 sb = *reinterpret_cast<const float4*>(&columns[(wn * S::TN + i) * 32 + q * 8 + lhi * 4]);
                *reinterpret_cast<float4*>(&park[l32 * PLD + i * 32 + q * 8 + lhi * 4]) =
                    make_float4((float)total[i][j][4 * q] * sa * sb.x, (float)total[i][j][4 * q + 1] * sa * sb.y, (float)total[i][j][4 * q + 2] * sa * sb.z,
                                (float)total[i][j][4 * q + 3] * sa * sb.w);
            }
#pragma unroll
        for (int it = 0; it < TURNS; ++it) {
            const int id = it * WAVE + lane;
            const int64_t row = row0 + id / PIECES, col = ncol0 + id % PIECES * 8;
            const float4 low = *reinterpret_cast<const float4*>(&park[id / PIECES * PLD + id % PIECES * 8]), high = *reinterpret_cast<const float4*>(&park[id / PIECES * PLD + id % PIECES * 8 + 4]);
            if (row >= m_end || col >= p.n) continue;
            const float d[8] = {low.x, low.y, low.z, low.w, high.x, high.y, high.z, high.w};
            float gate[8], up[8];
            g[it].widen(gate);
            u[it].widen(up);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                float act, derivative;
                gate_math(p.activation, gate[e], act, derivative);
                gate[e] = d[e] * up[e] * derivative;
                up[e] = d[e] * act;
            }
            TO* dz = static_cast<TO*>(p.out) + row * p.ldo + col;
            if constexpr (sizeof(TO) == 4) {
#pragma unroll
                for (int e = 0; e < 8; e += 4) {
                    store_piece(dz + e, col + e, p.n, make_uint4(__float_as_uint(gate[e]), __float_as_uint(gate[e + 1]), __float_as_uint(gate[e + 2]), __float_as_uint(gate[e + 3])));
                    store_piece(dz + p.n + e, col + e, p.n, make_uint4(__float_as_uint(up[e]), __float_as_uint(up[e + 1]), __float_as_uint(up[e + 2]), __float_as_uint(up[e + 3])));
                }
            } else {
                uint32_t w[8];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    w[e] = narrow16<TO>(gate[2 * e]) | narrow16<TO>(gate[2 * e + 1]) << 16;
                    w[4 + e] = narrow16<TO>(up[2 * e]) | narrow16<TO>(up[2 * e + 1]) << 16;
                }
                store_piece(dz, col, p.n, make_uint4(w[0], w[1], w[2], w[3]));
                store_piece(dz + p.n, col, p.n, make_uint4(w[4], w[5], w[6], w[7]));
            }
        }
    }
}

constexpr int64_t GATED_MOST_K = 2048;

template <typename S> constexpr int int8_lds() { return S::STAGES * S::STAGE + 2 * S::COLS * 4; }

// Rows [m_begin, m_end) of one group and the columns from n_begin on.
template <typename S, bool GATED>
__device__ __forceinline__ void int8_tile(const Int8Args& p, int group, int64_t m_begin, int64_t m_end, int64_t n_begin, uint8_t* lds) {
    constexpr int TM = S::TM, TN = S::TN, STAGES = S::STAGES, RING = STAGES * S::STAGE, HALVES = S::HALVES;
    static_assert(S::TEAMS == 1);
    const int tid = threadIdx.x, lane = tid % WAVE, l32 = lane % 32, lhi = lane / 32;
    const int wave = __builtin_amdgcn_readfirstlane(tid / WAVE);
    const int wm = wave / S::WN, wn = wave % S::WN;
    float* columns = reinterpret_cast<float*>(lds + RING);                   // the channels' scales, then the bias
    if (tid < S::COLS) {
        const int64_t col = n_begin + tid;
        columns[tid] = !p.sb ? 1.0f : col < p.n ? p.sb[(int64_t)group * p.n + col] : 0.0f;
        columns[S::COLS + tid] = p.bias && col < p.n ? load_float(p.bias, col, p.bias_dtype) : -0.0f;   // adding -0 changes nothing
    }

    // ---- load plan: instruction `it` brings LOAD_ROWS rows of an operand, unit U = PIECES row + slot holds piece slot ^ swizzle(row)
    const i32x4 res_a = raw_resource(p.a + m_begin * p.lda), res_b = raw_resource(p.b + (int64_t)group * p.b_stride + n_begin * p.ldb);
    constexpr uint32_t OUTSIDE = 0x80000000u;
    const int chunks = (int)((p.k + S::CHUNK - 1) / S::CHUNK), full_chunks = (int)(p.k / S::CHUNK);
    auto swizzle = [](int row) -> int { return S::PIECES == 4 ? (row >> 2) & 3 : (row >> 1) & 7; };
    const int piece = tid % S::PIECES ^ swizzle(tid / S::PIECES);
    const bool inside_tail = (int64_t)full_chunks * S::CHUNK + piece * 16 < p.k;
    uint32_t cur[S::LOADS];
#pragma unroll
    for (int it = 0; it < S::LOADS; ++it) {
        const int r = (it < S::A_LOADS ? it : it - S::A_LOADS) * S::LOAD_ROWS + tid / S::PIECES;
        const int64_t rows = it < S::A_LOADS ? m_end - m_begin : p.n - n_begin;
        cur[it] = (uint32_t)(r < rows ? r : rows - 1) * (uint32_t)(it < S::A_LOADS ? p.lda : p.ldb) + piece * 16;
    }
    const uint32_t lds_base = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint8_t*)lds;
    auto issue = [&](int c, int stage) {
        if (__builtin_expect(c >= full_chunks, 0)) {                         // the chunk that straddles the end of k, and those past it
            asm volatile("; end of the k range");
            const bool here = c == full_chunks && inside_tail;
#pragma unroll
            for (int it = 0; it < S::LOADS; ++it) {
                const uint32_t at = here ? cur[it] : OUTSIDE;
                load16_to_lds(it < S::A_LOADS ? res_a : res_b, lds_base + (uint32_t)stage * S::STAGE + it * 8192 + (uint32_t)wave * 1024, at, (uint32_t)c * S::CHUNK);
            }
            return;
        }
#pragma unroll
        for (int it = 0; it < S::LOADS; ++it)
            load16_to_lds(it < S::A_LOADS ? res_a : res_b, lds_base + (uint32_t)stage * S::STAGE + it * 8192 + (uint32_t)wave * 1024, cur[it], (uint32_t)c * S::CHUNK);
    };

    // ---- operand reads
    const int sw = swizzle(l32);
    const int rd_a0 = (wm * TM * 32 + l32) * S::CHUNK + ((lhi ^ sw) * 16), rd_b0 = S::A_BYTES + (wn * TN * 32 + l32) * S::CHUNK + ((lhi ^ sw) * 16);
    i32x16 total[TN][TM];
#pragma unroll
    for (int i = 0; i < TN; ++i)
#pragma unroll
        for (int j = 0; j < TM; ++j)
#pragma unroll
            for (int r = 0; r < 16; ++r) total[i][j][r] = 0;
    i32x4 oa[HALVES][TM][2], ob[HALVES][TN][2];                              // 32 k each
    auto read = [&](int stage) {
        const uint8_t* base = lds + stage * S::STAGE;
        int rd_a = rd_a0, rd_b = rd_b0;
        asm volatile("" : "+v"(rd_a), "+v"(rd_b));                           // the addresses below: formed anew, 256 x 256 has no registers to keep them
#pragma unroll
        for (int h = 0; h < HALVES; ++h)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
#pragma unroll
                for (int i = 0; i < TN; ++i) ob[h][i][e] = *reinterpret_cast<const i32x4*>(base + ((rd_b + i * 32 * S::CHUNK) ^ (h * 64 + e * 32)));
#pragma unroll
                for (int j = 0; j < TM; ++j) oa[h][j][e] = *reinterpret_cast<const i32x4*>(base + ((rd_a + j * 32 * S::CHUNK) ^ (h * 64 + e * 32)));
            }
    };
    auto math = [&] {
        __builtin_amdgcn_s_setprio(1);
#pragma unroll
        for (int h = 0; h < HALVES; ++h)
#pragma unroll
            for (int e = 0; e < 2; ++e)
#pragma unroll
                for (int i = 0; i < TN; ++i)
#pragma unroll
                    for (int j = 0; j < TM; ++j) total[i][j] = __builtin_amdgcn_mfma_i32_32x32x32_i8(ob[h][i][e], oa[h][j][e], total[i][j], 0, 0, 0);
        // (the compiler sinks MFMAs into the following read phase otherwise: intrinsics without side effects cross a barrier)
#pragma unroll
        for (int i = 0; i < TN; ++i)
#pragma unroll
            for (int j = 0; j < TM; ++j) asm volatile("" : "+v"(total[i][j]));
        __builtin_amdgcn_s_setprio(0);
    };
    auto pin_operands = [&] {                                                // in registers before the barrier
#pragma unroll
        for (int h = 0; h < HALVES; ++h)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
#pragma unroll
                for (int j = 0; j < TM; ++j) asm volatile("" : "+v"(oa[h][j][e]));
#pragma unroll
                for (int i = 0; i < TN; ++i) asm volatile("" : "+v"(ob[h][i][e]));
            }
    };
    auto barrier = [] {
        __builtin_amdgcn_sched_barrier(0);
        asm volatile("s_barrier" ::: "memory");
        __builtin_amdgcn_sched_barrier(0);
    };

    // Phases as in pingpong_tile (gemm_pingpong.hpp): waves 0-3 read chunk c in phase 2c and multiply in phase 2c + 1, waves 4-7 one phase later; the loads of
    // chunk c + STAGES - 1 go into the stage of chunk c - 1, whose last readers had their operands in registers before the barrier that ended
    // their phase; every wave ends its read phase of chunk c with its own loads of chunk c + 1 landed. Two stages: chunk c + 1 goes out once
    // waves 4-7 have read chunk c - 1, and every wave waits for its part before the barrier that ends phase 2c + 1.
    constexpr bool TWO = STAGES == 2;
    constexpr int AHEAD = TWO ? 0 : (STAGES - 2) * S::LOADS;
    static_assert((STAGES - 1) * S::LOADS < 16);
#pragma unroll
    for (int s = 0; s < (TWO ? 2 : STAGES - 1); ++s) issue(s, s);
    __builtin_amdgcn_s_waitcnt(0x0F70 | (TWO ? S::LOADS : AHEAD));           // chunk 0
    barrier();
    const bool late = wave >= 4;
    if (late) barrier();
    int stage = 0, fill = TWO && late ? 0 : STAGES - 1;
    for (int c = 0; c < chunks; ++c) {
        read(stage);
        auto issue_next = [&](int next) {
            if (!TWO || next > 1) issue(next, fill);                         // (two stages: chunk 1 went out with chunk 0)
            fill = fill == STAGES - 1 ? 0 : fill + 1;
        };
        if (!TWO || !late) issue_next(c + STAGES - 1);
        stage = stage == STAGES - 1 ? 0 : stage + 1;
        __builtin_amdgcn_sched_barrier(0);
        if (!TWO || late) __builtin_amdgcn_s_waitcnt(0x0070 | AHEAD);
        else __builtin_amdgcn_s_waitcnt(0xC07F);                             // the LDS reads alone
        pin_operands();
        barrier();
        if (TWO && late) issue_next(c + 2);
        math();
        if (TWO && !late) __builtin_amdgcn_s_waitcnt(0x0F70);
        barrier();
    }
    if (!late) barrier();
    __builtin_amdgcn_s_waitcnt(0x0F70);                                      // the trailing loads must not land in what follows
    __syncthreads();                                                         // every wave has left the ring, and the columns' scales are there
    if constexpr (GATED) {
        if (p.out_dtype == VIOLA_F32) store_int8_gradient<S, float>(total, p, m_begin, m_end, n_begin, lds, columns);
        else if (p.out_dtype == VIOLA_BF16) store_int8_gradient<S, bf16_t>(total, p, m_begin, m_end, n_begin, lds, columns);
        else store_int8_gradient<S, f16_t>(total, p, m_begin, m_end, n_begin, lds, columns);
    } else if (p.out_dtype == VIOLA_F32) store_int8_tile<S>(total, p, static_cast<float*>(p.out), m_begin, m_end, n_begin, lds, columns);
    else if (p.out_dtype == VIOLA_BF16) store_int8_tile<S>(total, p, static_cast<bf16_t*>(p.out), m_begin, m_end, n_begin, lds, columns);
    else store_int8_tile<S>(total, p, static_cast<f16_t*>(p.out), m_begin, m_end, n_begin, lds, columns);
}

// Rows that no group has, of one tile
template <typename S, typename TO> __device__ __forceinline__ void int8_zeros(const Int8Args& p, int64_t m_begin, int64_t m_end, int64_t n_begin, int64_t shift) {
    constexpr int PER = 16 / (int)sizeof(TO), PIECES = S::COLS / PER;
    for (int i = threadIdx.x; i < S::ROWS * PIECES; i += S::THREADS) {
        const int64_t row = m_begin + i / PIECES, col = n_begin + i % PIECES * PER;
        if (row < m_end && col < p.n) store_piece(static_cast<TO*>(p.out) + row * p.ldo + shift + col, col, p.n, make_uint4(0, 0, 0, 0));
    }
}

template <typename S, int WAVES_PER_SIMD, bool GATED> __global__ __launch_bounds__(512, WAVES_PER_SIMD) void int8_gemm(Int8Args p) {
    __shared__ __attribute__((aligned(1024))) uint8_t lds[int8_lds<S>()];
    // contiguous ranges for each XCD, of the tiles that there are: the host knows a bound on those of groups
    const int tiles_m = p.offsets ? int8_count_tiles(p, S::ROWS) : p.tiles_m, each = (tiles_m * p.tiles_n + 7) / 8;
    const int t = blockIdx.x % 8 * each + blockIdx.x / 8;
    if ((int)blockIdx.x / 8 >= each || t >= tiles_m * p.tiles_n) return;
    // groups of 8 row tiles, as in pingpong_place
    const int across = 8 * p.tiles_n, first_m = t / across * 8;
    const int rows_here = tiles_m - first_m < 8 ? tiles_m - first_m : 8;
    const int64_t n_begin = (int64_t)(t % across / rows_here) * S::COLS;
    int group;
    int64_t m_begin, m_end;
    if (!int8_row_tile(p, first_m + t % across % rows_here, S::ROWS, group, m_begin, m_end)) return;
    if (!p.offsets || group < p.groups) int8_tile<S, GATED>(p, group, m_begin, m_end, n_begin, lds);
    else
        for (int64_t half = 0; half < (GATED ? 2 : 1); ++half) {             // (zero is zero in either type of 16 bits)
            if (p.out_dtype == VIOLA_F32) int8_zeros<S, float>(p, m_begin, m_end, n_begin, half * p.n);
            else int8_zeros<S, bf16_t>(p, m_begin, m_end, n_begin, half * p.n);
        }
}

// 256 x 256 in four stages of 64 k, or in two of 128 k for long sums (16384 x 4096 -> 11008 668 and 690 us, 32768 rows at 16 experts of 4096 -> 1024 165 and 185, 4096 x 11008 -> 4096
// 161 and 153)
using Int8L = PingPongShape<2, 4, 4, 2, 4>;
using Int8Long = PingPongShape<2, 4, 4, 2, 2, 128>;
using Int8M = PingPongShape<4, 2, 2, 2, 3, 128>;                             // 256 x 128
using Int8S = PingPongShape<2, 4, 2, 1, 3, 128>;                             // 128 x 128
using Int8Pairs = PingPongShape<2, 4, 2, 1, 4>;                              // 128 x 128, two blocks on a CU
using Int8Wide = PingPongShape<4, 2, 2, 2, 3>;                               // 256 x 128, two blocks on a CU

template <typename S, int WAVES_PER_SIMD, bool GATED = false> static int launch_tiles(const Int8Args& args, hipStream_t stream) {
    Int8Args p = args;
    const int64_t tiles_m = int8_row_tiles(p, S::ROWS), tiles_n = (p.n + S::COLS - 1) / S::COLS;
    if (tiles_m * tiles_n >= (int64_t{1} << 32) / 512 - 8) return VIOLA_ETOOLARGE;                // threads of a grid
    p.tiles_m = (int)tiles_m;
    p.tiles_n = (int)tiles_n;
    const dim3 grid((unsigned)((tiles_m * tiles_n + 7) / 8 * 8));
    VIOLA_LAUNCH((int8_gemm<S, WAVES_PER_SIMD, GATED>), grid, 512, 0, stream, p);
    return viola_launch_status();
}

// The tile that takes least by estimates in microseconds, fitted to measured times of 30 shapes and within 15 % of most. A round of a tile for each CU takes a fixed part and a time
// for each chunk of 64 k, which grows with the share of CUs at work as the clock falls: L .42 to .84 + 9.5, M .30 to .47 + 6.3, S .24 to .29 + 4, two S on a CU .25 to
// .73 + 4, two M 1 to 1.04 + 6.4 (one's ends under the other's products, slower ones: for short sums). Each group leaves half a row tile unfilled on average. So
// 8192 x 1024 -> 4096 takes L (47 us; M 57, S 66), 8192 x 4096 -> 1024 M (35; L 49, S 47), 2048 x 2048 -> 2048 S (13; M 17), 9850 x 770 -> 1000 L (18; M 25), 4000 rows at 128
// experts of 2048 -> 1024 pairs of S (61; L 69), 16384 x 512 -> 2048 pairs of M (28; L 33, pairs of S 34).
enum Int8TileShape { INT8_L, INT8_M, INT8_S, INT8_PAIRS, INT8_WIDE };
static Int8TileShape choose_int8_tile(const Int8Args& p) {
    const double chunks = (double)((p.k + 63) / 64);
    auto estimate = [&](int rows, int cols, int at_once, double idle, double busy, double fixed) {
        const int64_t row_tiles = (p.m + rows - 1) / rows + (p.offsets ? (p.groups < p.m ? p.groups : p.m) / 2 : 0), tiles = row_tiles * ((p.n + cols - 1) / cols);
        const double full = (double)(tiles / at_once), rest = (double)(tiles % at_once) / at_once;
        return full * (chunks * busy + fixed) + (rest > 0 ? chunks * (idle + (busy - idle) * rest) + fixed : 0.0);
    };
    const double time[5] = {estimate(256, 256, 256, 0.42, 0.84, 9.5), estimate(256, 128, 256, 0.30, 0.47, 6.3), estimate(128, 128, 256, 0.24, 0.29, 4.0),
                            estimate(128, 128, 512, 0.25, 0.73, 4.0), estimate(256, 128, 512, 1.0, 1.04, 6.4)};
    int best = 0;
    for (int i = 1; i < 5; ++i) best = time[i] < time[best] ? i : best;
    return (Int8TileShape)best;
}

static int launch_int8(const Int8Args& p, hipStream_t stream) {
    if (p.z) return launch_tiles<Int8Pairs, 4, true>(p, stream);
    if (int8_rows_fit(p)) return launch_int8_rows(p, stream);
    switch (choose_int8_tile(p)) {
        case INT8_L: return p.k > 8192 ? launch_tiles<Int8Long, 2>(p, stream) : launch_tiles<Int8L, 2>(p, stream);
        case INT8_M: return launch_tiles<Int8M, 2>(p, stream);
        case INT8_S: return launch_tiles<Int8S, 2>(p, stream);
        case INT8_WIDE: return launch_tiles<Int8Wide, 4>(p, stream);
        default: return launch_tiles<Int8Pairs, 4>(p, stream);
    }
}

}  // namespace viola

using namespace viola;

namespace {

int product(Int8Args p, int64_t groups, hipStream_t stream) {
    VIOLA_CHECK_ARG(p.m >= 0 && p.n > 0 && p.k > 0 && p.m < (int64_t{1} << 31) && p.n < (int64_t{1} << 30) && groups >= 0 && viola_is_float(p.out_dtype) &&
                    (!p.bias || viola_is_float(p.bias_dtype)) && (!p.offsets || (groups > 0 && !p.bias)));
    if (p.k > INT8_MOST_K || groups > INT8_MOST_GROUPS) return VIOLA_EUNSUPPORTED;
    if (p.m == 0) return 0;
    VIOLA_CHECK_ARG(p.a && p.sa && p.b && p.out && p.lda >= p.k && p.ldb >= p.k && p.lda % 16 == 0 && p.ldb % 16 == 0 && p.lda <= 2 * INT8_MOST_K && p.b_stride % 16 == 0 &&
                    reinterpret_cast<uintptr_t>(p.a) % 16 == 0 && reinterpret_cast<uintptr_t>(p.b) % 16 == 0);
    if (p.ldb > (int64_t{1} << 22)) return VIOLA_EUNSUPPORTED;               // rows of one tile within 32 bits
    p.k = (p.k + 15) / 16 * 16;
    p.groups = (int)groups;
    return launch_int8(p, stream);
}

}  // namespace

extern "C" int viola_int8_gemm(const int8_t* a, int64_t lda, const float* sa, const int8_t* b, int64_t ldb, int64_t b_stride, const float* sb, const int32_t* offsets,
                               int64_t groups, int64_t m, int64_t n, int64_t k, const void* bias, int bias_dtype, void* out, int out_dtype, viola_stream_t stream_) {
    hipStream_t stream = viola_enter(stream_);
    Int8Args p = {};
    p.a = a; p.b = b; p.sa = sa; p.sb = sb; p.bias = bias; p.out = out; p.m = m; p.n = n; p.k = k;
    p.lda = lda; p.ldb = ldb; p.ldo = n; p.offsets = offsets; p.b_stride = b_stride; p.bias_dtype = bias_dtype; p.out_dtype = out_dtype;
    return product(p, groups, stream);
}

extern "C" int viola_int8_gemm_gated_backward(const int8_t* a, int64_t lda, const float* sa, const int8_t* b, int64_t ldb, int64_t b_stride, const int32_t* offsets,
                                              int64_t groups, int64_t m, int64_t n, int64_t k, const void* z, int64_t z_pitch, int z_dtype, int activation, void* dz,
                                              viola_stream_t stream_) {
    hipStream_t stream = viola_enter(stream_);
    VIOLA_CHECK_ARG(activation >= 0 && activation <= VIOLA_RELU && m >= 0 && n > 0 && z_pitch >= 2 * n);
    Int8Args p = {};
    p.a = a; p.b = b; p.sa = sa; p.out = dz; p.m = m; p.n = n; p.k = k; p.lda = lda; p.ldb = ldb; p.ldo = 2 * n; p.offsets = offsets; p.b_stride = b_stride;
    p.out_dtype = z_dtype; p.z = z; p.z_pitch = z_pitch; p.activation = activation;
    if (m == 0 && viola_is_float(z_dtype)) return 0;
    VIOLA_CHECK_ARG(z);
    p.groups = groups > 0 && groups <= INT8_MOST_GROUPS ? (int)groups : 1;
    if (int8_rows_fit(p) || k > GATED_MOST_K) return VIOLA_EUNSUPPORTED;      // two calls
    return product(p, groups, stream);
}
