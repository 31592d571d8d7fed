// Rows in 8-bit integers with a scale each, and the gradient through a gated activation: what stands around the products of int8_gemm.hip.
//
//   quantize   s = max_c |v_c| / 127 (rounded to 32 bits), q_c = v_c / s rounded to the nearest integer, a half to the even one
//              v = x, or act(g) u of a row [g | u], or x times a factor for each column (a product's channel scales, in its backward pass)
//   backward   dz = [dh u act'(g) | dh act(g)] with dh in 32 bits
//
// A row of zeros has s = 0 and zeros; a row that holds an Inf or a NaN has s = NaN and zeros, so a product makes all of it NaN and no other row. Where s is
// subnormal the quotient may pass 127 and is cut off there.
//
// The integer is that of the exact quotient: v times the reciprocal is within 2^-14 of it, which settles all but the neighbourhood of a half; there the
// residual v - q s, one fused operation without error where it is near s / 2 (s and v are multiples of the smaller one's last place, which the result has
// 24 bits of), is compared with s / 2.
//
// Both are bound by memory: each value is read once and stays in registers between the maximum and the quotients. A wavefront has a row of up to 2048 values, four
// wavefronts one of up to 8192, eight one of up to 16384; longer rows are read twice.
#include "int8_quantize.hpp"

#include <type_traits>

using namespace viola;

namespace {

enum { PLAIN = 0, GATED = 1, SCALED = 2 };                                   // what is quantized: x, act(g) u, x times factors (with sums over the rows)

struct QuantizeArgs {
    const void* x;
    int64_t pitch, rows;                                                     // pitch in values
    int cols, activation, groups, whole;                                     // whole: x can be read eight values at a time
    const float* factors;                                                    // SCALED: [groups][cols]
    const int* offsets;                                                      // SCALED: where the rows of each group begin; null: one group
    int8_t* codes;
    int64_t code_pitch;                                                      // a multiple of 16; zeros past the columns
    float* scales;
    float* partial;                                                          // SCALED: [parts][cols] sums of x, null: not wanted
    int64_t per_block;                                                       // rows
    bool stream_in;
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

// What is quantized of a piece, of columns c to c + 7; raw: x itself
template <typename T, int MODE>
__device__ __forceinline__ void value8(const QuantizeArgs& a, const T* row, const float* factors, int c, float (&v)[8], float (&raw)[8]) {
    load8<T>(row, c, a.cols, a.whole, a.stream_in, v);
    if constexpr (MODE == GATED) {
        float u[8];
        load8<T>(row + a.cols, c, a.cols, a.whole, a.stream_in, u);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            float act, derivative;
            gate_math(a.activation, v[i], act, derivative);
            v[i] = act * u[i];
        }
    } else if constexpr (MODE == SCALED) {
        float f[8];
        load8<float>(factors, c, a.cols, a.cols % 4 == 0, false, f);         // rows of whole 16 bytes
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            raw[i] = v[i];
            v[i] *= f[i];
        }
    }
}

constexpr int threads_of(int waves) { return waves <= 4 ? 256 : 64 * waves; }

// A row of WAVES wavefronts, PIECES pieces of eight values a thread. SCALED: a block goes through per_block rows and leaves the sums of x
// over those of each of its rows of threads.
template <typename T, int MODE, int WAVES, int PIECES> __global__ __launch_bounds__(threads_of(WAVES)) void quantize_rows(QuantizeArgs a) {
    constexpr int THREADS = 64 * WAVES, TOGETHER = threads_of(WAVES) / THREADS;
    __shared__ uint32_t most_of[2][threads_of(WAVES) / 64];
    const int t = threadIdx.x % THREADS, slot = threadIdx.x / THREADS, wave = threadIdx.x / 64;
    const int64_t first = blockIdx.x * a.per_block, end = first + a.per_block < a.rows ? first + a.per_block : a.rows;
    float sums[MODE == SCALED ? PIECES : 1][8];
    if constexpr (MODE == SCALED)
#pragma unroll
        for (int p = 0; p < PIECES; ++p)
#pragma unroll
            for (int i = 0; i < 8; ++i) sums[p][i] = 0.0f;
    int turn = 0;
    for (int64_t row = first + slot; row - slot < end; row += TOGETHER) {
        const bool here = row < end;
        const T* x = static_cast<const T*>(a.x) + row * a.pitch;
        const float* factors = a.factors;
        if (MODE == SCALED && a.offsets && here) factors += (int64_t)group_of(a.offsets, a.groups, row) * a.cols;
        float v[PIECES][8];
        uint32_t most = 0;
#pragma unroll
        for (int p = 0; p < PIECES; ++p) {
            const int c = (p * THREADS + t) * 8;
#pragma unroll
            for (int i = 0; i < 8; ++i) v[p][i] = 0.0f;
            if (!here || c >= a.cols) continue;
            float raw[8];
            value8<T, MODE>(a, x, factors, c, v[p], raw);
            most = magnitudes(v[p], most);
            if constexpr (MODE == SCALED)
#pragma unroll
                for (int i = 0; i < 8; ++i) sums[p][i] += raw[i];
        }
        most = lanes_max<64>(most);
        if constexpr (WAVES > 1) {                                           // two sets of slots in turn: one barrier a row
            if (threadIdx.x % 64 == 0) most_of[turn][wave] = most;
            __syncthreads();
#pragma unroll
            for (int w = 0; w < WAVES; ++w) {
                const uint32_t other = most_of[turn][slot * WAVES + w];
                most = other > most ? other : most;
            }
            turn ^= 1;
        }
        if (!here) continue;
        const RowScale scale(most);
        if (t == 0) a.scales[row] = scale.s;
#pragma unroll
        for (int p = 0; p < PIECES; ++p) {
            const int c = (p * THREADS + t) * 8;
            if (c < a.code_pitch) *reinterpret_cast<uint2*>(a.codes + row * a.code_pitch + c) = encode8_int(v[p], scale);
        }
    }
    if constexpr (MODE == SCALED) {
        if (!a.partial) return;
        float* to = a.partial + (int64_t)(blockIdx.x * TOGETHER + slot) * a.cols;
#pragma unroll
        for (int p = 0; p < PIECES; ++p) {
            const int c = (p * THREADS + t) * 8;
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (c + i < a.cols) to[c + i] = sums[p][i];
        }
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
    auto factors_of = [&](int64_t row) { return MODE == SCALED && a.offsets ? a.factors + (int64_t)group_of(a.offsets, a.groups, row) * a.cols : a.factors; };
    for (int r = 0; r < rows; ++r) {
        const float* factors = factors_of(first + r);
        uint32_t most = 0;
        for (int c = t * 8; c < a.cols; c += 512 * 8) {
            float v[8], raw[8];
            value8<T, MODE>(a, static_cast<const T*>(a.x) + (first + r) * a.pitch, factors, c, v, raw);
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
            if (c < a.cols) value8<T, MODE>(a, static_cast<const T*>(a.x) + (first + r) * a.pitch, factors_of(first + r), c, v, raw);
            *reinterpret_cast<uint2*>(a.codes + (first + r) * a.code_pitch + c) = encode8_int(v, scale);
            if constexpr (MODE == SCALED)
#pragma unroll
                for (int i = 0; i < 8; ++i) sums[i] += raw[i];
        }
        if (MODE == SCALED && a.partial)
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (c + i < a.cols) a.partial[(int64_t)blockIdx.x * a.cols + c + i] = sums[i];
    }
}

// How rows are shared: wavefronts of a row, rows of a block, blocks, and rows of sums that they leave.
struct Shares {
    int waves, pieces;                                                       // 0 wavefronts: long rows
    int64_t per_block, blocks, parts;
};
Shares shares_of(int64_t rows, int64_t cols, bool sums) {
    Shares s = {};
    if (cols > 16384) {
        s.per_block = LONG_ROWS;
        s.blocks = (rows + LONG_ROWS - 1) / LONG_ROWS;
        s.parts = s.blocks;
        return s;
    }
    s.waves = cols <= 2048 ? 1 : cols <= 8192 ? 4 : 8;
    const int64_t piece = 512 * s.waves;                                     // values that the row's threads have at once
    s.pieces = cols <= piece ? 1 : cols <= 2 * piece ? 2 : 4;
    const int64_t together = s.waves == 1 ? 4 : 1;
    // sums: four blocks for each CU at most, a row of sums from each of a block's rows of threads
    s.per_block = together;
    if (sums && rows > 1024 * together) s.per_block = (rows + 1024 * together - 1) / (1024 * together) * together;
    s.blocks = (rows + s.per_block - 1) / s.per_block;
    s.parts = s.blocks * together;
    return s;
}

template <typename T, int MODE> int launch(QuantizeArgs& a, hipStream_t stream) {
    const Shares s = shares_of(a.rows, a.cols, a.partial != nullptr);
    a.per_block = s.per_block;
    if (s.blocks >= (int64_t{1} << 31)) return VIOLA_ETOOLARGE;
    const dim3 grid((unsigned)s.blocks);
    auto with = [&](auto waves, auto pieces) {
        constexpr int WAVES = decltype(waves)::value, PIECES = decltype(pieces)::value;
        VIOLA_LAUNCH((quantize_rows<T, MODE, WAVES, PIECES>), grid, threads_of(WAVES), 0, stream, a);
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
    int cols, activation, whole;
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
        load8<T>(z, c, a.cols, a.whole, false, g);
        load8<T>(z + a.cols, c, a.cols, a.whole, false, u);
        load8<float>(a.dh + row * a.cols, c, a.cols, a.whole, false, d);
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

bool readable8(const void* x, int64_t pitch, int64_t cols, int dtype, bool halves) {
    const int unit = 16 / viola_dtype_size(dtype);
    return reinterpret_cast<uintptr_t>(x) % 16 == 0 && pitch % unit == 0 && (!halves || cols % unit == 0);
}

}  // namespace

extern "C" int64_t viola_int8_sum_parts(int64_t rows, int64_t cols) { return rows <= 0 || cols <= 0 ? 0 : shares_of(rows, cols, true).parts; }

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
    a.whole = readable8(x, pitch, cols, dtype, gated);
    a.stream_in = false;
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
    a.whole = readable8(z, pitch, cols, dtype, true) && cols % 4 == 0 && reinterpret_cast<uintptr_t>(dz) % 16 == 0 && reinterpret_cast<uintptr_t>(dh) % 16 == 0;
    const int64_t blocks = (rows * ((cols + 7) / 8) + 255) / 256;
    const dim3 grid((unsigned)(blocks < 16384 ? blocks : 16384));
    if (dtype == VIOLA_F32) VIOLA_LAUNCH((gated_gradient_kernel<float>), grid, 256, 0, stream, a);
    else if (dtype == VIOLA_BF16) VIOLA_LAUNCH((gated_gradient_kernel<bf16_t>), grid, 256, 0, stream, a);
    else VIOLA_LAUNCH((gated_gradient_kernel<f16_t>), grid, 256, 0, stream, a);
    return viola_launch_status();
}
