// Rows in 8-bit integers with a scale each, and the gradient through a gated activation: what stands around the products of int8_gemm.hip.
//
//   quantize   s = max_c |v_c| / 127 (rounded to 32 bits), q_c = v_c / s rounded to the nearest integer, a half to the even one
//              v = x, or act(g) u of a row [g | u], or x times a factor for each column (a product's channel scales, in its backward pass)
//   backward   dz = [dh u act'(g) | dh act(g)] with dh in 32 bits
//
// A row of zeros has s = 0 and zeros; a row that holds an Inf or a NaN has s = NaN and zeros, so a product makes all of it NaN and no other row. Where s is
// subnormal the quotient may pass 127 and is cut off there.
//
// The integer is that of the exact quotient: v times the reciprocal is within 2^-17 of it (127 times half a last place), which settles all but 2 10^-5 around a half; there the
// residual v - q s, one fused operation without error where it is near s / 2 (s and v are multiples of the smaller one's last place, which the result has
// 24 bits of), is compared with s / 2.
//
// Both are bound by memory: each value is read once and stays in registers between the maximum and the quotients. A wavefront has a row of up to 2048 values, four
// wavefronts one of up to 8192, eight one of up to 16384; longer rows are read twice.
// bf16, us: 8192 x 1024 8.5, 16384 x 4096 31 (6.5 TB/s read and written), 4096 x 11008 gated 40 (5.6); times factors with sums 8192 x 4096 25, without 32768 x 1024 23.
#include "int8_quantize.hpp"

#include <type_traits>

using namespace viola;

namespace {

enum { PLAIN = 0, GATED = 1, SCALED = 2 };                                   // what is quantized: x, act(g) u, x times factors (with sums over the rows)

struct QuantizeArgs {
    const void* x;
    int64_t pitch, rows;                                                     // pitch in values
    int cols, activation, groups;
    const float* factors;                                                    // SCALED: [groups][cols]
    const int* offsets;                                                      // SCALED: where the rows of each group begin; null: one group
    int8_t* codes;
    int64_t code_pitch;                                                      // a multiple of 16; zeros past the columns
    float* scales;
    float* partial;                                                          // SCALED: [parts][cols] sums of x, null: not wanted
    int64_t per_block;                                                       // rows
};

// The group whose rows `row` is among (the last one for rows behind all of them, which no product reads).
__device__ __forceinline__ int group_of(const int* offsets, int groups, int64_t row) {
    int low = 0, high = groups - 1;
    while (low < high) {
        const int middle = (low + high + 1) / 2;
        if (offsets[middle] <= row) low = middle;
        else high = middle - 1;
    }
    return low;
}

// What is quantized of columns c to c + 7
template <typename T, int MODE> __device__ __forceinline__ void value8(const QuantizeArgs& a, const T* row, int c, float (&v)[8]) {
    load8<T>(row, c, a.cols, v);
    if constexpr (MODE == GATED) {
        float u[8];
        load8<T>(row + a.cols, c, a.cols, u);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            float act, derivative;
            gate_math(a.activation, v[i], act, derivative);
            v[i] = act * u[i];
        }
    }
}

typedef float loose_floats4 __attribute__((ext_vector_type(4), aligned(4)));
__device__ __forceinline__ void store_sums(float* to, int c, int cols, const float (&sums)[8]) {
    if (c + 8 <= cols) {
        *reinterpret_cast<loose_floats4*>(to + c) = loose_floats4{sums[0], sums[1], sums[2], sums[3]};
        *reinterpret_cast<loose_floats4*>(to + c + 4) = loose_floats4{sums[4], sums[5], sums[6], sums[7]};
        return;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i)
        if (c + i < cols) to[c + i] = sums[i];
}

constexpr int threads_of(int waves) { return waves <= 4 ? 256 : 64 * waves; }

// The largest magnitude of a row of WAVES wavefronts, in all of them: two sets of slots in turn, so one barrier a row is enough
template <int WAVES> __device__ __forceinline__ uint32_t over_row(uint32_t most, uint32_t (*slots)[threads_of(WAVES) / 64], int& turn) {
    most = lanes_max<64>(most);
    if constexpr (WAVES > 1) {
        if (threadIdx.x % 64 == 0) slots[turn][threadIdx.x / 64] = most;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < WAVES; ++w) {
            const uint32_t other = slots[turn][threadIdx.x / 64 / WAVES * WAVES + w];
            most = other > most ? other : most;
        }
        turn ^= 1;
    }
    return most;
}

// A row of WAVES wavefronts, PIECES pieces of eight values a thread.
template <typename T, int MODE, int WAVES, int PIECES> __global__ __launch_bounds__(threads_of(WAVES)) void quantize_rows(QuantizeArgs a) {
    constexpr int THREADS = 64 * WAVES, TOGETHER = threads_of(WAVES) / THREADS;
    __shared__ uint32_t slots[2][threads_of(WAVES) / 64];
    const int t = threadIdx.x % THREADS;
    const int64_t row = ((int64_t)blockIdx.y * gridDim.x + blockIdx.x) * TOGETHER + threadIdx.x / THREADS;
    const bool here = row < a.rows;
    float v[PIECES][8];
    uint32_t most = 0;
#pragma unroll
    for (int p = 0; p < PIECES; ++p) {
        const int c = (p * THREADS + t) * 8;
#pragma unroll
        for (int i = 0; i < 8; ++i) v[p][i] = 0.0f;
        if (!here || c >= a.cols) continue;
        value8<T, MODE>(a, static_cast<const T*>(a.x) + row * a.pitch, c, v[p]);
        most = magnitudes(v[p], most);
    }
    int turn = 0;
    most = over_row<WAVES>(most, slots, turn);
    if (!here) return;
    const RowScale scale(most);
    if (t == 0) a.scales[row] = scale.s;
#pragma unroll
    for (int p = 0; p < PIECES; ++p) {
        const int c = (p * THREADS + t) * 8;
        if (c < a.code_pitch) *reinterpret_cast<uint2*>(a.codes + row * a.code_pitch + c) = encode8_int(v[p], scale);
    }
}

// x times factors: a block goes through per_block rows, the next one's loads under the work on each, with the factors of their group in registers, and leaves the sums
// of x over its rows (SUMS).
template <typename T, int WAVES, int PIECES, bool SUMS> __global__ __launch_bounds__(threads_of(WAVES)) void quantize_scaled_rows(QuantizeArgs a) {
    constexpr int THREADS = 64 * WAVES, TOGETHER = threads_of(WAVES) / THREADS;
    __shared__ uint32_t slots[2][threads_of(WAVES) / 64];
    __shared__ __attribute__((aligned(16))) float others[SUMS && TOGETHER > 1 ? (TOGETHER - 1) * PIECES * THREADS * 8 : 4];
    const int t = threadIdx.x % THREADS, slot = threadIdx.x / THREADS;
    const int64_t first = blockIdx.x * a.per_block, end = first + a.per_block < a.rows ? first + a.per_block : a.rows;
    float sums[SUMS ? PIECES : 1][8], factor[PIECES][8];
    Raw8<T> next[PIECES];
    if constexpr (SUMS)
#pragma unroll
        for (int p = 0; p < PIECES; ++p)
#pragma unroll
            for (int i = 0; i < 8; ++i) sums[p][i] = 0.0f;
    auto load = [&](int64_t row) {                                           // (past the end: the last row once more)
        const T* x = static_cast<const T*>(a.x) + (row < end ? row : end - 1) * a.pitch;
#pragma unroll
        for (int p = 0; p < PIECES; ++p) {
            const int c = (p * THREADS + t) * 8;
            if (c < a.cols) next[p].load(x, c, a.cols);
        }
    };
    auto load_factors = [&](const float* factors) {
#pragma unroll
        for (int p = 0; p < PIECES; ++p) {
            const int c = (p * THREADS + t) * 8;
#pragma unroll
            for (int i = 0; i < 8; ++i) factor[p][i] = 0.0f;
            if (c < a.cols) load8<float>(factors, c, a.cols, factor[p]);
        }
    };
#pragma unroll
    for (int p = 0; p < PIECES; ++p) next[p].clear();
    load(first + slot);
    if (!a.offsets) load_factors(a.factors);
    int64_t until = -1;                                                      // rows that the factors are for
    int turn = 0;
    for (int64_t row = first + slot; row - slot < end; row += TOGETHER) {
        const bool here = row < end;
        if (a.offsets && here && row >= until) {                             // (one row for a wavefront or more: no lane of it goes another way)
            const int g = group_of(a.offsets, a.groups, row);
            until = g + 1 < a.groups ? a.offsets[g + 1] : a.rows;
            load_factors(a.factors + (int64_t)g * a.cols);
        }
        float v[PIECES][8];
        uint32_t most = 0;
#pragma unroll
        for (int p = 0; p < PIECES; ++p) {
            next[p].widen(v[p]);
            if (SUMS && here)
#pragma unroll
                for (int i = 0; i < 8; ++i) sums[p][i] += v[p][i];
#pragma unroll
            for (int i = 0; i < 8; ++i) v[p][i] *= factor[p][i];
            most = magnitudes(v[p], most);
        }
        load(row + TOGETHER);
        most = over_row<WAVES>(most, slots, turn);
        if (!here) continue;
        const RowScale scale(most);
        if (t == 0) a.scales[row] = scale.s;
#pragma unroll
        for (int p = 0; p < PIECES; ++p) {
            const int c = (p * THREADS + t) * 8;
            if (c < a.code_pitch) *reinterpret_cast<uint2*>(a.codes + row * a.code_pitch + c) = encode8_int(v[p], scale);
        }
    }
    if constexpr (SUMS) {                                                    // the rows of threads of a block in order
        if constexpr (TOGETHER > 1) {
            if (slot)
#pragma unroll
                for (int p = 0; p < PIECES; ++p)
#pragma unroll
                    for (int i = 0; i < 8; i += 4)
                        *reinterpret_cast<float4*>(&others[((slot - 1) * PIECES + p) * THREADS * 8 + t * 4 + i * THREADS]) =
                            make_float4(sums[p][i], sums[p][i + 1], sums[p][i + 2], sums[p][i + 3]);
            __syncthreads();
            if (slot) return;
#pragma unroll
            for (int s = 0; s < TOGETHER - 1; ++s)
#pragma unroll
                for (int p = 0; p < PIECES; ++p)
#pragma unroll
                    for (int i = 0; i < 8; i += 4) {
                        const float4 more = *reinterpret_cast<const float4*>(&others[(s * PIECES + p) * THREADS * 8 + t * 4 + i * THREADS]);
                        sums[p][i] += more.x; sums[p][i + 1] += more.y; sums[p][i + 2] += more.z; sums[p][i + 3] += more.w;
                    }
        }
        float* to = a.partial + (int64_t)blockIdx.x * a.cols;
#pragma unroll
        for (int p = 0; p < PIECES; ++p) store_sums(to, (p * THREADS + t) * 8, a.cols, sums[p]);
    }
}

// Rows that do not fit a block's registers: read twice, the second time piece after piece for all rows of the block, so that sums over the rows need
// one piece's registers.
constexpr int LONG_ROWS = 16;
template <typename T, int MODE> __global__ __launch_bounds__(512) void quantize_long_rows(QuantizeArgs a) {
    __shared__ uint32_t most_of[LONG_ROWS][8];
    const int t = threadIdx.x;
    const int64_t first = (int64_t)blockIdx.x * LONG_ROWS, left = a.rows - first;
    const int rows = left < LONG_ROWS ? (int)left : LONG_ROWS;
    auto value = [&](int r, int c, float (&v)[8], float (&raw)[8]) {
        value8<T, MODE>(a, static_cast<const T*>(a.x) + (first + r) * a.pitch, c, v);
        if constexpr (MODE == SCALED) {
            const float* factors = a.offsets ? a.factors + (int64_t)group_of(a.offsets, a.groups, first + r) * a.cols : a.factors;
            float f[8];
            load8<float>(factors, c, a.cols, f);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                raw[i] = v[i];
                v[i] *= f[i];
            }
        }
    };
    for (int r = 0; r < rows; ++r) {
        uint32_t most = 0;
        for (int c = t * 8; c < a.cols; c += 512 * 8) {
            float v[8], raw[8];
            value(r, c, v, raw);
            most = magnitudes(v, most);
        }
        most = lanes_max<64>(most);
        if (t % 64 == 0) most_of[r][t / 64] = most;
    }
    __syncthreads();
    for (int c = t * 8; c < a.code_pitch; c += 512 * 8) {
        float sums[8] = {};
        for (int r = 0; r < rows; ++r) {
            uint32_t most = most_of[r][0];
#pragma unroll
            for (int w = 1; w < 8; ++w) most = most_of[r][w] > most ? most_of[r][w] : most;
            const RowScale scale(most);
            if (c == 0) a.scales[first + r] = scale.s;
            float v[8] = {}, raw[8] = {};
            if (c < a.cols) value(r, c, v, raw);
            *reinterpret_cast<uint2*>(a.codes + (first + r) * a.code_pitch + c) = encode8_int(v, scale);
            if constexpr (MODE == SCALED)
#pragma unroll
                for (int i = 0; i < 8; ++i) sums[i] += raw[i];
        }
        if (MODE == SCALED && a.partial) store_sums(a.partial + (int64_t)blockIdx.x * a.cols, c, a.cols, sums);
    }
}

// How rows are shared: wavefronts of a row, rows of a block, blocks. x times factors: as many rows as leave 1024 blocks, or 512 where each leaves a row of sums
// (8192 x 4096: 21 us, 27 with 512 blocks; with sums and their reduction 30, 35 with 1024).
struct Shares {
    int waves, pieces;                                                       // 0 wavefronts: long rows
    int64_t per_block, blocks;
};
enum Purpose { ONCE, SCALE, SCALE_AND_SUM };
Shares shares_of(int64_t rows, int64_t cols, Purpose purpose) {
    Shares s = {};
    if (cols > 16384) {
        s.per_block = LONG_ROWS;
    } else {
        s.waves = cols <= 2048 ? 1 : cols <= 8192 ? 4 : 8;
        const int64_t piece = 512 * s.waves;                                 // values that the row's threads have at once
        s.pieces = cols <= piece ? 1 : cols <= 2 * piece ? 2 : 4;
        s.per_block = s.waves == 1 ? 4 : 1;
        const int64_t most = s.per_block * (purpose == SCALE ? 1024 : 512);
        if (purpose != ONCE && rows > most) s.per_block *= (rows + most - 1) / most;
    }
    s.blocks = (rows + s.per_block - 1) / s.per_block;
    return s;
}

constexpr int64_t MOST_ACROSS = 1 << 20;                                     // blocks in a row of the grid, which takes fewer than 2^32 threads
template <typename T, int MODE> int launch(QuantizeArgs& a, hipStream_t stream) {
    const Shares s = shares_of(a.rows, a.cols, MODE != SCALED ? ONCE : a.partial ? SCALE_AND_SUM : SCALE);
    a.per_block = s.per_block;
    if (s.blocks >= (int64_t{1} << 31)) return VIOLA_ETOOLARGE;
    const int64_t across = MODE == SCALED || s.waves == 0 || s.blocks < MOST_ACROSS ? s.blocks : MOST_ACROSS;
    const dim3 grid((unsigned)across, (unsigned)((s.blocks + across - 1) / across));
    auto with = [&](auto waves, auto pieces) {
        constexpr int WAVES = decltype(waves)::value, PIECES = decltype(pieces)::value;
        if constexpr (MODE != SCALED) VIOLA_LAUNCH((quantize_rows<T, MODE, WAVES, PIECES>), grid, threads_of(WAVES), 0, stream, a);
        else if (a.partial) VIOLA_LAUNCH((quantize_scaled_rows<T, WAVES, PIECES, true>), grid, threads_of(WAVES), 0, stream, a);
        else VIOLA_LAUNCH((quantize_scaled_rows<T, WAVES, PIECES, false>), grid, threads_of(WAVES), 0, stream, a);
    };
    using std::integral_constant;
    const int key = s.waves * 8 + s.pieces;
    if (s.waves == 0) VIOLA_LAUNCH((quantize_long_rows<T, MODE>), grid, 512, 0, stream, a);
    else if (key == 9) with(integral_constant<int, 1>(), integral_constant<int, 1>());
    else if (key == 10) with(integral_constant<int, 1>(), integral_constant<int, 2>());
    else if (key == 12) with(integral_constant<int, 1>(), integral_constant<int, 4>());
    else if (key == 34) with(integral_constant<int, 4>(), integral_constant<int, 2>());
    else if (key == 36) with(integral_constant<int, 4>(), integral_constant<int, 4>());
    else with(integral_constant<int, 8>(), integral_constant<int, 4>());
    return viola_launch_status();
}
template <typename T> int launch_mode(QuantizeArgs& a, hipStream_t stream) {
    if (a.factors) return launch<T, SCALED>(a, stream);
    return a.activation >= 0 ? launch<T, GATED>(a, stream) : launch<T, PLAIN>(a, stream);
}

// ---------------------------------------------------------------------------------------------------- gated activation, backward
struct GatedGradientArgs {
    const void* z;
    const float* dh;
    void* dz;
    const int* total;                                                        // rows in use, on the device; null: all
    int64_t pitch, rows;
    int cols, activation, whole;                                             // whole: rows of dz are of whole 16 bytes
};

template <typename T> __device__ __forceinline__ void store8(T* to, int n, bool whole, const float (&v)[8]) {
    if (whole) {
        if constexpr (sizeof(T) == 4) {
            reinterpret_cast<float4*>(to)[0] = make_float4(v[0], v[1], v[2], v[3]);
            reinterpret_cast<float4*>(to)[1] = make_float4(v[4], v[5], v[6], v[7]);
        } else {
            uint32_t w[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) w[i] = narrow16<T>(v[2 * i]) | narrow16<T>(v[2 * i + 1]) << 16;
            *reinterpret_cast<uint4*>(to) = make_uint4(w[0], w[1], w[2], w[3]);
        }
        return;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i)
        if (i < n) to[i] = from_f32<T>(v[i]);
}

template <typename T> __global__ __launch_bounds__(256) void gated_gradient_kernel(GatedGradientArgs a) {
    const int pieces = (a.cols + 7) / 8;
    const int64_t total = a.rows * pieces, used = a.total ? *a.total : a.rows;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
        const int64_t row = i / pieces;
        const int c = (int)(i - row * pieces) * 8;
        const T* z = static_cast<const T*>(a.z) + row * a.pitch;
        float g[8], u[8], d[8];
        load8<T>(z, c, a.cols, g);
        load8<T>(z + a.cols, c, a.cols, u);
        load8<float>(a.dh + row * a.cols, c, a.cols, d);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            float act, derivative;
            gate_math(a.activation, g[j], act, derivative);
            g[j] = row < used ? d[j] * u[j] * derivative : 0.0f;
            u[j] = row < used ? d[j] * act : 0.0f;
        }
        T* dz = static_cast<T*>(a.dz) + row * 2 * a.cols;
        const bool whole = a.whole && c + 8 <= a.cols;
        store8<T>(dz + c, a.cols - c, whole, g);
        store8<T>(dz + a.cols + c, a.cols - c, whole, u);
    }
}

}  // namespace

extern "C" int64_t viola_int8_sum_parts(int64_t rows, int64_t cols) { return rows <= 0 || cols <= 0 ? 0 : shares_of(rows, cols, SCALE_AND_SUM).blocks; }

extern "C" int viola_int8_quantize(const void* x, int64_t pitch, int dtype, int64_t rows, int64_t cols, int activation, const float* factors, const int32_t* offsets,
                                   int64_t groups, int8_t* codes, int64_t code_pitch, float* scales, float* partial, viola_stream_t stream_) {
    hipStream_t stream = viola_enter(stream_);
    const bool gated = activation >= 0;
    VIOLA_CHECK_ARG(viola_is_float(dtype) && rows >= 0 && cols > 0 && cols <= (int64_t{1} << 28) && activation <= VIOLA_RELU && pitch >= (gated ? 2 : 1) * cols);
    VIOLA_CHECK_ARG(code_pitch >= cols && code_pitch % 16 == 0 && code_pitch < cols + 16 && !(factors && gated) && (factors || (!offsets && !partial)) && groups >= (offsets ? 1 : 0));
    if (rows == 0) return 0;
    VIOLA_CHECK_ARG(x && codes && scales && reinterpret_cast<uintptr_t>(codes) % 16 == 0 && reinterpret_cast<uintptr_t>(factors) % 16 == 0 &&
                    reinterpret_cast<uintptr_t>(scales) % 4 == 0);
    QuantizeArgs a = {};
    a.x = x; a.pitch = pitch; a.rows = rows; a.cols = (int)cols; a.activation = activation; a.groups = (int)groups; a.factors = factors; a.offsets = offsets;
    a.codes = codes; a.code_pitch = code_pitch; a.scales = scales; a.partial = partial;
    if (dtype == VIOLA_F32) return launch_mode<float>(a, stream);
    return dtype == VIOLA_BF16 ? launch_mode<bf16_t>(a, stream) : launch_mode<f16_t>(a, stream);
}

extern "C" int viola_int8_gated_backward(const void* z, int64_t pitch, int dtype, int64_t rows, int64_t cols, int activation, const float* dh, const int32_t* total,
                                         void* dz, viola_stream_t stream_) {
    hipStream_t stream = viola_enter(stream_);
    VIOLA_CHECK_ARG(viola_is_float(dtype) && rows >= 0 && cols > 0 && cols <= (int64_t{1} << 28) && activation >= 0 && activation <= VIOLA_RELU && pitch >= 2 * cols);
    if (rows == 0) return 0;
    VIOLA_CHECK_ARG(z && dh && dz);
    GatedGradientArgs a = {};
    a.z = z; a.dh = dh; a.dz = dz; a.total = total; a.pitch = pitch; a.rows = rows; a.cols = (int)cols; a.activation = activation;
    a.whole = reinterpret_cast<uintptr_t>(dz) % 16 == 0 && cols % (16 / viola_dtype_size(dtype)) == 0;
    const int64_t blocks = (rows * ((cols + 7) / 8) + 255) / 256;
    const dim3 grid((unsigned)(blocks < 16384 ? blocks : 16384));
    if (dtype == VIOLA_F32) VIOLA_LAUNCH((gated_gradient_kernel<float>), grid, 256, 0, stream, a);
    else if (dtype == VIOLA_BF16) VIOLA_LAUNCH((gated_gradient_kernel<bf16_t>), grid, 256, 0, stream, a);
    else VIOLA_LAUNCH((gated_gradient_kernel<f16_t>), grid, 256, 0, stream, a);
    return viola_launch_status();
}
