// The norms before and after a block with its gate and residual sum: what the kernels of norm.hip compute.
//
//   n(v) = (v - mu) r,  r = (mean((v - mu)^2) + eps)^-1/2,  mu = mean(v), or 0 for the root mean square
//   after the block   x' = rho x + alpha g (n(y) w_a + b_a)         (or n(y) = y)
//   before the next   h  = (n(x') w_b + b_b) (1 + s) + t
//
// Backward, from D_out = dL/dx' and dh, with x' computed again in 32 bits from x and y (as many bytes as reading x' would be, without its
// rounding):
//   q = dh w_b (1 + s),  D = D_out + r_x (q - x^ mean(q x^) - mean(q)),  dx = rho D,  p = D alpha g w_a,
//   dy = r_y (p - y^ mean(p y^) - mean(p))
// with x^ = (x' - mu_x) r_x and y^ alike (the means without a product only with mu). Sums over rows: A1 = sum D y^, A0 = sum D, S1 = sum dh x^, S0 = sum dh give every
// vector's gradient: dw_a = alpha sum g A1, db_a = alpha sum g A0, dg = alpha (w_a A1 + b_a A0), dw_b = sum (1 + s) S1,
// db_b = sum (1 + s) S0, ds = w_b S1 + b_b S0, dt = S0.
#pragma once

#include "block_ops.hpp"

#include <type_traits>

namespace viola {

// FORM_PLAIN: FORM_BETWEEN without a norm, weight or bias after the block: x' = rho x + alpha g y
enum { FORM_BEFORE = 0, FORM_AFTER = 1, FORM_BETWEEN = 2, FORM_PLAIN = 3 };
enum { SUM_A1 = 1, SUM_A0 = 2, SUM_S1 = 4, SUM_S0 = 8 };

// A vector along the row: one for all rows (pitch 0), or one for each group of rows.
struct NormVector {
    const void* data;
    int64_t pitch;
};

struct NormArgs {
    const void *x, *y;
    int64_t x_pitch, y_pitch, rows, group_rows;
    int cols, x_dtype, branch_dtype, after, before, weight_dtype, vector_dtype;
    const void *after_weight, *after_bias, *weight, *bias;
    NormVector gate, scale, shift;
    float rho, alpha, eps;
    // forward
    void *out, *h;
    float4* stats;                                                           // mu_y, r_y, mu_x, r_x of a row
    int64_t chunk;                                                           // rows of a block
    int team;                                                                // threads of a row, where rows are in registers
    bool stream_in, stream_out;                                              // rows are read, written past the caches' order
    // backward
    const void *dout, *dh;
    void *dx, *dy;
    float* parts;                                                            // [portions][sums][cols]
    int64_t portions, per_group;                                             // portions in all, and of one group
    int sums;                                                                // which sums over rows are wanted (SUM_*)
};

// ---------------------------------------------------------------------------------------------------- rows in registers
// A row belongs to a team of whole wavefronts, eight elements to a thread, from its loads to its stores: each tensor is read once and written
// once whatever the norms in between need. A block has several teams where rows are narrow; they take its rows in turn. The vectors along
// the row are kept folded for the rows of a group: x' = rho x + y^ GA + GB with GA = alpha g w_a, GB = alpha g b_a, and h = x^ W + B with
// W = w_b (1 + s), B = b_b (1 + s) + t. BIAS: GB and A0 are there, SHIFT: S0 is; most norms
// do without them and their registers.
//
// Bound by memory: two or three reads and two writes an element against some 40 operations. Forward and backward between two blocks, cold caches: 16384 rows
// of 4096 in bf16 104 and 161 us (5.2 and 5.0 TB/s, what a large copy reaches here), 16384 rows of 1152 with a gate, a scale and a shift for each of 64 images 35
// and 49 us (4.2 and 4.6: 16 of 64 lanes of a row's third wavefront have work, and 128 registers leave the backward pass four wavefronts a SIMD).
// Eight elements a thread are one load of 16 bytes from a 16-bit tensor, and leave registers for the next rows' loads under way.
// x' is computed twice and not stored in 32 bits between the passes: its reading would cost what x and y cost.
constexpr int ROW_THREADS = 1024, ROW_COLUMNS = 8 * ROW_THREADS;

// The type of rows that are no whole aligned pieces: any of the three, known when they are read. A thread then has the elements `step` apart from its
// first on, so that a wavefront's access is of neighbours.
struct loose_t {};

template <typename T> struct Piece { uint4 word[sizeof(T) / 2]; };           // eight elements as they lie in memory
template <> struct Piece<loose_t> { float value[8]; };

// A thread's elements of a row: eight from `col` on, or `count` of them `step` apart.
struct Place {
    uint32_t col, step;
    int count;
    __device__ __forceinline__ Place(const NormArgs& a, int t, int threads, bool loose) : col(loose ? t : 8 * t), step(loose ? threads : 1) {
        const int left = a.cols - (int)col;
        count = left <= 0 ? 0 : loose ? min((left + threads - 1) / threads, 8) : 8;
    }
    __device__ __forceinline__ bool any() const { return count > 0; }
    __device__ __forceinline__ uint32_t column(int i) const { return col + i * step; }
};

// Streamed or not (block_ops.hpp); 32-bit pieces never are: an access of a wavefront is every other 16 bytes of them, which streamed fill no line
// (4 x 2048 rows of 2048 on a 32-bit stream: 56 instead of 45 us).
// `row` elements behind `base` for a whole wavefront, `col` more for a thread: the first is a scalar's work, the second an offset of 32 bits.
template <typename T, bool STREAM> __device__ __forceinline__ Piece<T> load_piece(const void* base, int64_t row, const Place& at, int dtype) {
    if constexpr (__is_same(T, loose_t)) {
        Piece<T> p = {};
        auto from = [&](auto type) {
            using U = decltype(type);
            const char* line = static_cast<const char*>(base) + row * (int64_t)sizeof(U);
            uint32_t offset = at.col * (uint32_t)sizeof(U);
            asm volatile("" : "+v"(offset));                                 // or eight of them for each tensor stay in registers from row to row
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (i < at.count) p.value[i] = to_f32(*reinterpret_cast<const U*>(line + (offset + i * at.step * (uint32_t)sizeof(U))));
        };
        if (dtype == VIOLA_F32) from(float());
        else if (dtype == VIOLA_BF16) from(bf16_t());
        else from(f16_t());
        return p;
    } else {
        const char* line = static_cast<const char*>(base) + row * (int64_t)sizeof(T);
        const uint4* from = reinterpret_cast<const uint4*>(line + at.col * (uint32_t)sizeof(T));
        Piece<T> p;
#pragma unroll
        for (int i = 0; i < (int)(sizeof(T) / 2); ++i) p.word[i] = load16<STREAM && sizeof(T) == 2>(from + i);
        return p;
    }
}
template <typename T> __device__ __forceinline__ void widen_piece(const Piece<T>& p, float (&v)[8]) {
    if constexpr (__is_same(T, loose_t)) {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = p.value[i];
    } else if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            v[4 * i] = __uint_as_float(p.word[i].x); v[4 * i + 1] = __uint_as_float(p.word[i].y);
            v[4 * i + 2] = __uint_as_float(p.word[i].z); v[4 * i + 3] = __uint_as_float(p.word[i].w);
        }
    } else {
        const uint32_t w[4] = {p.word[0].x, p.word[0].y, p.word[0].z, p.word[0].w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if constexpr (__is_same(T, bf16_t)) {
                v[2 * i] = __uint_as_float(w[i] << 16);
                v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
            } else {
                v[2 * i] = widen16<f16_t>(w[i] & 0xffffu);
                v[2 * i + 1] = widen16<f16_t>(w[i] >> 16);
            }
        }
    }
}
template <typename T> __device__ __forceinline__ void store_piece(void* base, int64_t row, const Place& at, int dtype, const float (&v)[8], bool stream) {
    char* line = static_cast<char*>(base) + row * (int64_t)sizeof(T);
    uint4* to = reinterpret_cast<uint4*>(line + at.col * (uint32_t)sizeof(T));
    if constexpr (__is_same(T, loose_t)) {
        auto to_line = [&](auto type) {
            using U = decltype(type);
            char* out = static_cast<char*>(base) + row * (int64_t)sizeof(U);
            uint32_t offset = at.col * (uint32_t)sizeof(U);
            asm volatile("" : "+v"(offset));
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (i < at.count) *reinterpret_cast<U*>(out + (offset + i * at.step * (uint32_t)sizeof(U))) = from_f32<U>(v[i]);
        };
        if (dtype == VIOLA_F32) to_line(float());
        else if (dtype == VIOLA_BF16) to_line(bf16_t());
        else to_line(f16_t());
    } else if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int i = 0; i < 2; ++i)
            store16(to + i, make_uint4(__float_as_uint(v[4 * i]), __float_as_uint(v[4 * i + 1]), __float_as_uint(v[4 * i + 2]), __float_as_uint(v[4 * i + 3])), false);
    } else if constexpr (__is_same(T, bf16_t)) {
        store16(to, make_uint4(f32_to_bf16x2_bits(v[0], v[1]), f32_to_bf16x2_bits(v[2], v[3]), f32_to_bf16x2_bits(v[4], v[5]), f32_to_bf16x2_bits(v[6], v[7])), stream);
    } else {
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = narrow16<f16_t>(v[2 * i]) | narrow16<f16_t>(v[2 * i + 1]) << 16;
        store16(to, make_uint4(w[0], w[1], w[2], w[3]), stream);
    }
}

// A thread's elements of a vector of any type, as they lie in memory: 32 bytes, or 16 and nothing. Loose ones are loaded when they are widened, one vector after
// the other: together they would take every register.
template <bool LOOSE> struct VectorPiece {
    uint4 word[2] = {};
    int64_t row = 0;
    __device__ __forceinline__ void load(const void* base, int64_t begin, const Place& at, int dtype) {
        row = begin;
        if (LOOSE || !base || !at.any()) return;
        const char* line = static_cast<const char*>(base) + (dtype == VIOLA_F32 ? row * 4 : row * 2);
        const uint4* from = reinterpret_cast<const uint4*>(line + (dtype == VIOLA_F32 ? at.col * 4 : at.col * 2));
        word[0] = from[0];
        if (dtype == VIOLA_F32) word[1] = from[1];
    }
    __device__ __forceinline__ void widen(const void* base, const Place& at, int dtype, float absent, float (&v)[8]) const {
        if (!base || !at.any()) {
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = absent;
        } else if constexpr (LOOSE) {
            widen_piece(load_piece<loose_t, false>(base, row, at, dtype), v);
            __builtin_amdgcn_sched_barrier(0);
        } else if (dtype == VIOLA_F32) {
            widen_piece(Piece<float>{{word[0], word[1]}}, v);
        } else if (dtype == VIOLA_BF16) {
            widen_piece(Piece<bf16_t>{{word[0]}}, v);
        } else {
            widen_piece(Piece<f16_t>{{word[0]}}, v);
        }
    }
};

// Sums over the wavefronts of a team of up to 16, in all of its threads: each wavefront's own in LDS, two sets of slots in turn (see
// BlockSums), and from there in the 16 lanes of a row at once. All teams of a block call it alike.
struct TeamSums {
    float2* slot;                                                            // two sets of 16 in LDS
    int waves, wave, mine, turn = 0;
    __device__ __forceinline__ TeamSums(float2* slot, int waves) : slot(slot), waves(waves), wave(threadIdx.x / 64) {
        const int other = threadIdx.x % 16;
        mine = other < waves ? wave / waves * waves + other : -1;            // whose sum this lane fetches
    }
    static __device__ __forceinline__ float over_row(float v) {
        v = dpp_add<0xB1>(v);
        v = dpp_add<0x4E>(v);
        v = dpp_add<0x141>(v);
        return dpp_add<0x140>(v);
    }
    __device__ __forceinline__ float2 both(float a, float b) {
        a = wave_total(a);
        b = wave_total(b);
        if (waves == 1) return make_float2(a, b);
        if (threadIdx.x % 64 == 0) slot[turn * 16 + wave] = make_float2(a, b);
        __syncthreads();
        const float2 v = mine < 0 ? make_float2(0.0f, 0.0f) : slot[turn * 16 + mine];
        turn ^= 1;
        return make_float2(over_row(v.x), over_row(v.y));
    }
    __device__ __forceinline__ float one(float a) {
        a = wave_total(a);
        if (waves == 1) return a;
        if (threadIdx.x % 64 == 0) slot[turn * 16 + wave].x = a;
        __syncthreads();
        const float v = mine < 0 ? 0.0f : slot[turn * 16 + mine].x;
        turn ^= 1;
        return over_row(v);
    }
    // s / n for inverse = 1 / n, but for the last place
    static __device__ __forceinline__ float quotient(float s, float n, float inverse) {
        const float near = s * inverse;
        return fmaf(fmaf(-near, n, s), inverse, near);
    }
    // The mean of a row and the sum of squares around it: each wavefront around its own mean first, those then moved to the row's. A row far from
    // zero keeps its digits, and the team meets once. columns: of the row, of which a wavefront has up to 512.
    __device__ __forceinline__ float2 around_mean(const float (&v)[8], bool in, int columns, float inverse) {
        const int here = columns - (wave % waves) * 512, other = columns - (threadIdx.x % 16) * 512;
        float s = 0.0f, q = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; ++i) s += v[i];
        s = wave_total(in ? s : 0.0f);
        const float mean = s * __builtin_amdgcn_rcpf((float)(here < 512 ? here : 512));      // any value near it serves
#pragma unroll
        for (int i = 0; i < 8; ++i) q = fmaf(v[i] - mean, v[i] - mean, q);
        q = wave_total(in ? q : 0.0f);
        if (waves == 1) {
            const float exact = quotient(s, (float)columns, inverse), off = exact - mean;
            return make_float2(exact, q - (float)columns * off * off);
        }
        if (threadIdx.x % 64 == 0) slot[turn * 16 + wave] = make_float2(s, q);
        __syncthreads();
        float2 w = mine < 0 ? make_float2(0.0f, 0.0f) : slot[turn * 16 + mine];
        turn ^= 1;
        const float row_mean = quotient(over_row(w.x), (float)columns, inverse);
        if (mine >= 0) {
            const float n = (float)(other < 512 ? other : 512), near = w.x * __builtin_amdgcn_rcpf(n);
            // around `near`, which is the wavefront's mean but for its last digits, and from there around the row's
            const float off = near - row_mean;
            w.y += n * off * off + 2.0f * off * fmaf(-n, near, w.x);
        }
        return make_float2(row_mean, over_row(w.y));
    }
};

// v^-1/2 within an ulp; the hardware's root reads what is below the normal numbers as zero.
__device__ __forceinline__ float inverse_root(float v) { return v < 1e-30f ? 1.0f / sqrtf(v) : __builtin_amdgcn_rsqf(v); }

template <bool LAYER, bool LOOSE>
__device__ __forceinline__ float2 row_statistics(const float (&v)[8], const Place& at, int kind, int columns, float inverse, float eps, TeamSums& sums) {
    float mean = 0.0f, q = 0.0f;                                             // columns beyond the row are zero, or their thread has none
    if (LAYER && kind == VIOLA_NORM_LAYER) {
        if constexpr (!LOOSE) {
            const float2 around = sums.around_mean(v, at.any(), columns, inverse);
            return make_float2(around.x, inverse_root(around.y * inverse + eps));
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) mean += v[i];
        mean = TeamSums::quotient(sums.one(mean), (float)columns, inverse);
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float d = LOOSE ? (i < at.count ? v[i] - mean : 0.0f) : v[i];
        q = fmaf(d, d, q);
    }
    return make_float2(mean, inverse_root(sums.one(at.any() ? q : 0.0f) * inverse + eps));
}

// All loads are under way before the first is used: a block waits for them once.
template <int FORM, bool LOOSE> struct NormVectors {
    float ga[8], gb[8], w[8], b[8];
    __device__ __forceinline__ void load(const NormArgs& a, int64_t group, Place at) {
        asm volatile("" : "+v"(at.col));                                     // or the addresses are kept in registers from group to group
        VectorPiece<LOOSE> gate, after_weight, after_bias, weight, bias, scale, shift;
        if constexpr (FORM == FORM_PLAIN) gate.load(a.gate.data, group * a.gate.pitch, at, a.vector_dtype);
        if constexpr (FORM == FORM_AFTER || FORM == FORM_BETWEEN) {
            after_weight.load(a.after_weight, 0, at, a.weight_dtype);
            after_bias.load(a.after_bias, 0, at, a.weight_dtype);
            gate.load(a.gate.data, group * a.gate.pitch, at, a.vector_dtype);
        }
        if constexpr (FORM != FORM_AFTER) {
            weight.load(a.weight, 0, at, a.weight_dtype);
            bias.load(a.bias, 0, at, a.weight_dtype);
            scale.load(a.scale.data, group * a.scale.pitch, at, a.vector_dtype);
            shift.load(a.shift.data, group * a.shift.pitch, at, a.vector_dtype);
        }
        __builtin_amdgcn_sched_barrier(0);
        float u[8];
        if constexpr (FORM == FORM_PLAIN) {
            gate.widen(a.gate.data, at, a.vector_dtype, 1.0f, ga);
#pragma unroll
            for (int i = 0; i < 8; ++i) ga[i] *= a.alpha;
        }
        if constexpr (FORM == FORM_AFTER || FORM == FORM_BETWEEN) {
            after_weight.widen(a.after_weight, at, a.weight_dtype, 1.0f, ga);
            after_bias.widen(a.after_bias, at, a.weight_dtype, 0.0f, gb);
            gate.widen(a.gate.data, at, a.vector_dtype, 1.0f, u);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                ga[i] *= a.alpha * u[i];
                gb[i] *= a.alpha * u[i];
            }
        }
        if constexpr (FORM != FORM_AFTER) {
            weight.widen(a.weight, at, a.weight_dtype, 1.0f, w);
            bias.widen(a.bias, at, a.weight_dtype, 0.0f, b);
            scale.widen(a.scale.data, at, a.vector_dtype, 0.0f, u);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                w[i] = fmaf(w[i], u[i], w[i]);
                b[i] = fmaf(b[i], u[i], b[i]);
            }
            shift.widen(a.shift.data, at, a.vector_dtype, 0.0f, u);
#pragma unroll
            for (int i = 0; i < 8; ++i) b[i] += u[i];
        }
        if constexpr (LOOSE) {                                               // columns beyond the row weigh nothing
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                if (i < at.count) continue;
                if constexpr (FORM != FORM_BEFORE) ga[i] = gb[i] = 0.0f;
                if constexpr (FORM != FORM_AFTER) w[i] = b[i] = 0.0f;
            }
        }
    }
};

// The rows [blockIdx.x chunk, + chunk), a team each in turn. Every team makes as many turns as the first, so that barriers meet.
// LAYER: one of the norms subtracts a mean; without it the kinds are known to be the root mean square.
template <typename TX, typename TY, int FORM, bool LAYER> __global__ __launch_bounds__(ROW_THREADS) void norm_forward_kernel(NormArgs a) {
    __shared__ float2 slots[32];
    const int threads = a.team, teams = blockDim.x / threads, team = __builtin_amdgcn_readfirstlane(threadIdx.x / threads), t = threadIdx.x - team * threads;
    TeamSums sums(slots, threads / 64);
    constexpr bool LOOSE = __is_same(TX, loose_t);
    const Place at(a, t, threads, LOOSE);
    const bool in = at.any();
    const float inverse = 1.0f / (float)a.cols;
    const int64_t begin = blockIdx.x * a.chunk, end = begin + a.chunk < a.rows ? begin + a.chunk : a.rows;
    NormVectors<FORM, LOOSE> vectors;
    int64_t group_end = -1;                                                  // of the rows that the vectors are those of
    // Two rows are under way while one is worked on; zero beyond the row.
    Piece<TX> raw_x = {}, next_x = {};
    Piece<TY> raw_y = {}, next_y = {};
    auto load = [&](int64_t row, Piece<TX>& to_x, Piece<TY>& to_y) {
        if (!in || row >= end) return;                                       // beyond the end: some row before, which nobody stores
        auto from = [&](auto stream) {
            to_x = load_piece<TX, decltype(stream)::value>(a.x, row * a.x_pitch, at, a.x_dtype);
            if constexpr (FORM != FORM_BEFORE) to_y = load_piece<TY, decltype(stream)::value>(a.y, row * a.y_pitch, at, a.branch_dtype);
        };
        a.stream_in ? from(std::true_type()) : from(std::false_type());
    };
    if constexpr (!LOOSE) {
        load(begin + team, raw_x, raw_y);
        load(begin + team + teams, next_x, next_y);
    }
    for (int64_t base = begin; base < end; base += teams) {
        const int64_t row = base + team;
        const bool there = in && row < end;
        if (row >= group_end && row < end) {
            const int64_t group = row / a.group_rows;
            group_end = (group + 1) * a.group_rows;
            vectors.load(a, group, at);
        }
        float x[8], y[8];
        if constexpr (LOOSE) load(row, raw_x, raw_y);                        // eight loads for each of them: no registers for more
        widen_piece(raw_x, x);
        if constexpr (FORM != FORM_BEFORE) widen_piece(raw_y, y);
        if constexpr (!LOOSE) {
            raw_x = next_x;
            raw_y = next_y;
            load(row + 2 * teams, next_x, next_y);
        }
        float4 stat = make_float4(0.0f, 1.0f, 0.0f, 1.0f);
        if constexpr (FORM == FORM_PLAIN) {
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] = fmaf(a.rho, x[i], y[i] * vectors.ga[i]);
        } else if constexpr (FORM != FORM_BEFORE) {
            if (a.after != VIOLA_NORM_NONE) {
                const float2 s = row_statistics<LAYER, LOOSE>(y, at, a.after, a.cols, inverse, a.eps, sums);
                stat.x = s.x;
                stat.y = s.y;
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] = fmaf(a.rho, x[i], fmaf((LAYER ? y[i] - stat.x : y[i]) * stat.y, vectors.ga[i], vectors.gb[i]));
        }
        if constexpr (FORM != FORM_BEFORE && LOOSE) {
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] = i < at.count ? x[i] : 0.0f;
        }
        if constexpr (FORM != FORM_BEFORE)
            if (there) store_piece<TX>(a.out, row * a.cols, at, a.x_dtype, x, a.stream_out);
        if constexpr (FORM != FORM_AFTER) {
            const float2 s = row_statistics<LAYER, LOOSE>(x, at, a.before, a.cols, inverse, a.eps, sums);
            stat.z = s.x;
            stat.w = s.y;
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] = fmaf((LAYER ? x[i] - s.x : x[i]) * s.y, vectors.w[i], vectors.b[i]);
            if (there) store_piece<TY>(a.h, row * a.cols, at, a.branch_dtype, x, a.stream_out);
        }
        if (a.stats && t == 0 && row < end) a.stats[row] = stat;
    }
}

// One portion: rows of one group, a team each in turn. The teams' sums are joined in LDS at the end, team by team.
template <typename TX, typename TY, int FORM, bool LAYER, bool BIAS, bool SHIFT> __global__ __launch_bounds__(ROW_THREADS) void norm_backward_kernel(NormArgs a) {
    __shared__ float2 slots[32];
    using Sum = std::conditional_t<__is_same(TX, loose_t), loose_t, float>;
    extern __shared__ float joined[];                                        // [teams - 1][cols] where a block has several teams
    const int threads = a.team, teams = blockDim.x / threads, team = __builtin_amdgcn_readfirstlane(threadIdx.x / threads), t = threadIdx.x - team * threads;
    TeamSums sums(slots, threads / 64);
    constexpr bool LOOSE = __is_same(TX, loose_t);
    const Place at(a, t, threads, LOOSE);
    const bool in = at.any();
    const float inverse = 1.0f / (float)a.cols;
    const int64_t length = (a.group_rows + a.per_group - 1) / a.per_group;
    for (int64_t portion = blockIdx.x; portion < a.portions; portion += gridDim.x) {
        const int64_t group = portion / a.per_group, group_end = (group + 1) * a.group_rows;
        const int64_t begin = group * a.group_rows + portion % a.per_group * length;
        const int64_t end = begin + length < group_end ? begin + length : group_end;
        NormVectors<FORM, LOOSE> vectors;                                           // its b is not used, and neither is gb without BIAS
        vectors.load(a, group, at);
        float a1[8] = {}, a0[8] = {}, s1[8] = {}, s0[8] = {};
        // Beyond the row and beyond the portion everything is zero, the row's statistics too, and stays zero: nothing below asks again.
        Piece<TX> raw_x = {}, raw_dout = {};
        Piece<TY> raw_y = {}, raw_dh = {};
        auto load = [&](int64_t row) {
            if (row < end) {
                if (!in) return;
                auto from = [&](auto stream) {
                    constexpr bool STREAM = decltype(stream)::value;
                    if constexpr (FORM != FORM_AFTER) raw_x = load_piece<TX, STREAM>(a.x, row * a.x_pitch, at, a.x_dtype);
                    if constexpr (FORM != FORM_BEFORE) raw_y = load_piece<TY, STREAM>(a.y, row * a.y_pitch, at, a.branch_dtype);
                    if constexpr (FORM != FORM_AFTER) raw_dh = load_piece<TY, STREAM>(a.dh, row * a.cols, at, a.branch_dtype);
                    if constexpr (FORM != FORM_BEFORE) if (a.dout) raw_dout = load_piece<TX, STREAM>(a.dout, row * a.cols, at, a.x_dtype);
                };
                a.stream_in ? from(std::true_type()) : from(std::false_type());
            } else {
                raw_x = raw_dout = {};
                raw_y = raw_dh = {};
            }
        };
        if constexpr (!LOOSE) load(begin + team);
        for (int64_t base = begin; base < end; base += teams) {
            const int64_t row = base + team;
            const bool there = in && row < end;
            if constexpr (LOOSE) load(row);
            float4 stat = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            if (there) stat = a.stats[row];
            float x[8], y[8], d[8], q[8];                                    // x^, y^, D, dh W
            if constexpr (FORM != FORM_BEFORE) {
                widen_piece(raw_y, y);
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    if constexpr (FORM != FORM_PLAIN) y[i] = (LAYER ? y[i] - stat.x : y[i]) * stat.y;
                    if constexpr (LOOSE) y[i] = i < at.count ? y[i] : 0.0f;
                }
            }
            if constexpr (FORM != FORM_AFTER) {
                widen_piece(raw_x, x);
                widen_piece(raw_dh, q);
            }
            const Piece<TX> dout = raw_dout;
            if constexpr (!LOOSE) load(row + teams);
            if constexpr (FORM != FORM_BEFORE) widen_piece(dout, d);
            if constexpr (FORM != FORM_AFTER) {
                float along = 0.0f, total = 0.0f;
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    if constexpr (FORM == FORM_BETWEEN || FORM == FORM_PLAIN) x[i] = fmaf(a.rho, x[i], BIAS ? fmaf(y[i], vectors.ga[i], vectors.gb[i]) : y[i] * vectors.ga[i]);
                    x[i] = (LAYER ? x[i] - stat.z : x[i]) * stat.w;
                    if constexpr (LOOSE) x[i] = i < at.count ? x[i] : 0.0f;
                    s1[i] = fmaf(q[i], x[i], s1[i]);
                    if constexpr (SHIFT) s0[i] += q[i];
                    q[i] *= vectors.w[i];
                    along = fmaf(q[i], x[i], along);
                    if constexpr (LAYER) total += q[i];
                }
                float m1, m0 = 0.0f;
                if constexpr (LAYER) {
                    const float2 both = sums.both(along, total);
                    m1 = both.x * inverse;
                    m0 = a.before == VIOLA_NORM_LAYER ? both.y * inverse : 0.0f;
                } else {
                    m1 = sums.one(along) * inverse;
                }
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const float from_h = q[i] - (LAYER ? fmaf(x[i], m1, m0) : x[i] * m1);
                    d[i] = FORM == FORM_BEFORE ? stat.w * from_h : fmaf(stat.w, from_h, d[i]);
                }
            }
            if (a.dx && there) {
                if constexpr (FORM == FORM_BEFORE) {
                    store_piece<TX>(a.dx, row * a.cols, at, a.x_dtype, d, a.stream_out);
                } else {
#pragma unroll
                    for (int i = 0; i < 8; ++i) x[i] = a.rho * d[i];
                    store_piece<TX>(a.dx, row * a.cols, at, a.x_dtype, x, a.stream_out);
                }
            }
            if constexpr (FORM != FORM_BEFORE) {
                float along = 0.0f, total = 0.0f;
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    a1[i] = fmaf(d[i], y[i], a1[i]);
                    if constexpr (BIAS) a0[i] += d[i];
                    d[i] *= vectors.ga[i];
                    if constexpr (FORM != FORM_PLAIN) along = fmaf(d[i], y[i], along);
                    if constexpr (LAYER && FORM != FORM_PLAIN) total += d[i];
                }
                if (!a.dy) continue;
                if (FORM != FORM_PLAIN && a.after != VIOLA_NORM_NONE) {
                    float m1, m0 = 0.0f;
                    if constexpr (LAYER) {
                        const float2 both = sums.both(along, total);
                        m1 = both.x * inverse;
                        m0 = a.after == VIOLA_NORM_LAYER ? both.y * inverse : 0.0f;
                    } else {
                        m1 = sums.one(along) * inverse;
                    }
#pragma unroll
                    for (int i = 0; i < 8; ++i) d[i] = stat.y * (d[i] - (LAYER ? fmaf(y[i], m1, m0) : y[i] * m1));
                }
                if (there) store_piece<TY>(a.dy, row * a.cols, at, a.branch_dtype, d, a.stream_out);
            }
        }
        float* to = a.parts + portion * __popc(a.sums) * a.cols;
        auto write = [&](float (&v)[8]) {
            if (teams > 1) {
                __syncthreads();                                             // the sum before has been read
                if (team && in) store_piece<Sum>(joined, (int64_t)(team - 1) * a.cols, at, VIOLA_F32, v, false);
                __syncthreads();
                if (!team && in)
                    for (int u = 1; u < teams; ++u) {
#pragma unroll
                        for (int i = 0; i < 8; ++i)
                            if (i < at.count) v[i] += joined[(u - 1) * a.cols + at.column(i)];
                    }
            }
            if (!team && in) store_piece<Sum>(to, 0, at, VIOLA_F32, v, false);
            to += a.cols;
        };
        if (a.sums & SUM_A1) write(a1);
        if constexpr (BIAS) if (a.sums & SUM_A0) write(a0);
        if (a.sums & SUM_S1) write(s1);
        if constexpr (SHIFT) if (a.sums & SUM_S0) write(s0);
    }
}

}  // namespace viola
