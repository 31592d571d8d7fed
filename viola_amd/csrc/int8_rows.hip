// Products of 8-bit integers for few rows (a decoding step, experts with a handful of tokens): bound by one read of the weights, and below some 10 MB of them by the
// latency of a launch that reads anything at all. So weights go straight into registers: a wavefront has 16 NT channels and a share of k of its own, two 16-byte pieces of
// a channel for each lane and step of 128 k (a whole cache line of each channel), steps loaded ahead under the arithmetic, and the wavefronts that share a tile add up
// through LDS, which is exact. The rows' integers come from memory, or (FUSED) the block makes them of x in its first microsecond, while its first weights are on their way.
// 8 x 4096 -> 11008 12 to 13.5 us (3.4 to 3.8 TB/s), 256 rows at 64 experts of 4096 -> 2048 94 (5.7), 1 x 1024 -> 4096 4.6.
#include "int8_args.hpp"
#include "int8_quantize.hpp"

namespace viola {

typedef int i32x4_t __attribute__((ext_vector_type(4)));

constexpr int ROWS_WAVES = 4;
constexpr int FUSED_ROWS = 4;
struct FusedArgs {
    const void* x;
    int64_t pitch;
    int rows, cols, activation;
};

// A barrier for LDS alone: loads into registers stay under way (__syncthreads need not leave them so).
__device__ __forceinline__ void lds_barrier() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

// The quantizer of a block: rows are cut into parts of 512 values, eight for each lane, and the wavefronts take the parts in turn, FUSED_PIECES each at most. They are
// loaded before the first weights, so that those are not waited for. Every block makes all of them, so more rows, or wider ones, take longer than as two launches: us with 4096 channels,
// here and as two, 4 x 1024 6.7 and 8.0, 4 x 2048 8.5 and 10.4, 2 x 4096 12.0 and 11.0 (with 11008 14.7 and 15.8), 8 x 1024 8.1 and 8.3 (with 11008 11.9 and 9.6), 4 x 4096 17.0 and
// 11.2; with 1024 channels 16 x 256 9.5 and 7.9.
constexpr int FUSED_PIECES = 4;
inline bool fused_fits(int64_t rows, int64_t cols) { return rows <= FUSED_ROWS && cols % 16 == 0 && rows * ((cols + 511) / 512) <= ROWS_WAVES * FUSED_PIECES; }
template <typename T> struct FusedRows {
    float v[FUSED_PIECES][8];
    int parts;                                                               // of 512 values, a piece for each lane of a wavefront, that a row has

    __device__ __forceinline__ void load(const FusedArgs& f) {
        const int lane = threadIdx.x % WAVE, wave = threadIdx.x / WAVE;
        parts = (f.cols + 511) / 512;
#pragma unroll
        for (int i = 0; i < FUSED_PIECES; ++i) {
            const int slot = i * ROWS_WAVES + wave, row = slot / parts, c = (slot % parts * WAVE + lane) * 8;
#pragma unroll
            for (int e = 0; e < 8; ++e) v[i][e] = 0.0f;
            if (row < f.rows && c < f.cols) load8<T>(static_cast<const T*>(f.x) + row * f.pitch, c, f.cols, v[i]);
        }
    }
    // codes of all rows into LDS (rows `stride` bytes apart, zeros behind the columns, which are a multiple of 16) and their scales
    __device__ __forceinline__ void encode(const FusedArgs& f, int8_t* codes, int stride, float* scales) {
        __shared__ uint32_t most_of[FUSED_PIECES * ROWS_WAVES];
        const int lane = threadIdx.x % WAVE, wave = threadIdx.x / WAVE;
#pragma unroll
        for (int i = 0; i < FUSED_PIECES; ++i) {
            const int slot = i * ROWS_WAVES + wave, row = slot / parts, c = (slot % parts * WAVE + lane) * 8;
            if (row >= f.rows) break;
            if (f.activation >= 0 && c < f.cols) {
                float u[8];
                load8<T>(static_cast<const T*>(f.x) + row * f.pitch + f.cols, c, f.cols, u);
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    float act, derivative;
                    gate_math(f.activation, v[i][e], act, derivative);
                    v[i][e] = act * u[e];
                }
            }
            const uint32_t most = lanes_max<64>(magnitudes(v[i], 0));
            if (lane == 0) most_of[slot] = most;
        }
        for (int i = threadIdx.x; i < f.rows * 8; i += 64 * ROWS_WAVES)       // up to 112 bytes of a row
            if (f.cols + i % 8 * 16 + 16 <= stride) *reinterpret_cast<uint4*>(codes + i / 8 * stride + f.cols + i % 8 * 16) = make_uint4(0, 0, 0, 0);
        lds_barrier();
#pragma unroll
        for (int i = 0; i < FUSED_PIECES; ++i) {
            const int slot = i * ROWS_WAVES + wave, row = slot / parts, c = (slot % parts * WAVE + lane) * 8;
            if (row >= f.rows) break;
            uint32_t most = 0;
            for (int part = row * parts; part < (row + 1) * parts; ++part) most = most_of[part] > most ? most_of[part] : most;
            const RowScale scale(most);
            if (c == 0) scales[row] = scale.s;
            if (c < f.cols) *reinterpret_cast<uint2*>(codes + row * stride + c) = encode8_int(v[i], scale);
        }
        lds_barrier();
    }
};

// T: type of x (FUSED), or void. ks: wavefronts that share a tile's k.
template <int MT, int NT, typename T> __global__ __launch_bounds__(64 * ROWS_WAVES) void int8_rows(Int8Args p, FusedArgs f, int ks) {
    constexpr bool FUSED = !std::is_same<T, void>::value;
    constexpr int U = MT * NT <= 2 ? 4 : 2;                                  // steps loaded ahead
    extern __shared__ __attribute__((aligned(16))) uint8_t shared[];
    __shared__ float scales[FUSED_ROWS];
    i32x4_t* sums = reinterpret_cast<i32x4_t*>(shared);                      // [wave][tile][lane]
    int8_t* codes = reinterpret_cast<int8_t*>(shared) + ROWS_WAVES * MT * NT * WAVE * 16;
    const int lane = threadIdx.x % WAVE, l16 = lane & 15, quarter = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / WAVE), part = wave % ks;
    const int64_t n0 = ((int64_t)blockIdx.x * (ROWS_WAVES / ks) + wave / ks) * 16 * NT;
    const bool active = n0 < p.n;                                            // (every wave takes part in the barriers)
    int group = 0;
    int64_t m_begin, m_end;
    if (!int8_row_tile(p, blockIdx.y, 16 * MT, group, m_begin, m_end)) return;
    if (p.offsets && group == p.groups) {                                    // rows that no group has
        if (!active) return;
        const int64_t left = p.n - n0 < 16 * NT ? p.n - n0 : 16 * NT;
        for (int64_t row = m_begin + part; row < m_end; row += ks)
            for (int c = lane; c < left; c += WAVE) store_float(p.out, row * p.ldo + n0 + c, p.out_dtype, 0.0f);
        return;
    }
    const int steps = (int)((p.k + 127) / 128), begin = active ? steps * part / ks : 0, end = active ? steps * (part + 1) / ks : 0;
    const int8_t* w[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        const int64_t row = n0 + 16 * t + l16;
        w[t] = p.b + (int64_t)group * p.b_stride + (row < p.n ? row : p.n - 1) * p.ldb + quarter * 32;
    }
    // rows past the end are the last one again (their results go nowhere), pieces past k the first of the row, with zeros of x against them
    const int8_t* x[MT];
    const int stride = (steps * 128 + 16);                                   // of codes in LDS: rows 16 bytes apart in the banks
#pragma unroll
    for (int i = 0; i < MT; ++i) {
        const int64_t row = m_begin + 16 * i + l16 < m_end ? m_begin + 16 * i + l16 : m_end - 1;
        x[i] = (FUSED ? codes + row * stride : p.a + row * p.lda) + quarter * 32;
    }
    uint4 ring_w[U][NT][2], ring_x[U][FUSED ? 1 : MT][2];
    const uint4 zero = make_uint4(0, 0, 0, 0);
    auto load = [&](int u, int step) __attribute__((always_inline)) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int from = step * 128 + quarter * 32 + 16 * h < p.k ? step * 128 + 16 * h : -quarter * 32;         // k is of whole pieces
#pragma unroll
            for (int t = 0; t < NT; ++t) ring_w[u][t][h] = *reinterpret_cast<const uint4*>(w[t] + from);
            if constexpr (!FUSED)
#pragma unroll
                for (int i = 0; i < MT; ++i) ring_x[u][i][h] = *reinterpret_cast<const uint4*>(x[i] + from);
        }
    };
    FusedRows<typename std::conditional<FUSED, T, float>::type> rows_in;
    if constexpr (FUSED) rows_in.load(f);
#pragma unroll
    for (int u = 0; u < U; ++u)
        if (begin + u < end) load(u, begin + u);
    if constexpr (FUSED) rows_in.encode(f, codes, stride, scales);
    i32x4_t total[MT][NT];
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < NT; ++j) total[i][j] = i32x4_t{0, 0, 0, 0};
    for (int g = begin; g < end; g += U) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (g + u >= end) break;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
#pragma unroll
                for (int i = 0; i < MT; ++i) {
                    uint4 q;
                    if constexpr (FUSED) {
                        q = *reinterpret_cast<const uint4*>(x[i] + (g + u) * 128 + 16 * h);
                    } else {
                        q = ring_x[u][i][h];
                        if ((g + u) * 128 + quarter * 32 + 16 * h >= p.k) q = zero;
                    }
#pragma unroll
                    for (int j = 0; j < NT; ++j)
                        total[i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(__builtin_bit_cast(i32x4_t, ring_w[u][j][h]), __builtin_bit_cast(i32x4_t, q), total[i][j], 0, 0, 0);
                }
            }
            if (g + u + U < end) load(u, g + u + U);
        }
    }
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < NT; ++j) sums[(wave * MT * NT + i * NT + j) * WAVE + lane] = total[i][j];
    __syncthreads();
    if (!active) return;
    for (int tile = part; tile < MT * NT; tile += ks) {
        i32x4_t v = {0, 0, 0, 0};
        for (int i = 0; i < ks; ++i) v += sums[((wave - part + i) * MT * NT + tile) * WAVE + lane];
        // lane l: row l % 16, channels 4 (l / 16) .. + 3 of the tile
        const int64_t row = m_begin + tile / NT * 16 + l16, col = n0 + tile % NT * 16 + quarter * 4;
        if (row >= m_end || col >= p.n) continue;
        const RowFactor factor(FUSED ? scales[row] : p.sa[row]);
        float out[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int64_t c = col + r < p.n ? col + r : p.n - 1;
            out[r] = (float)v[r] * factor.s;
            if (p.sb) out[r] *= p.sb[(int64_t)group * p.n + c];
            out[r] = fmaf(out[r], factor.lift, p.bias ? load_float(p.bias, c, p.bias_dtype) : -0.0f);
        }
        const int64_t at = row * p.ldo + col;
        if (p.n % 4 == 0 && p.out_dtype == VIOLA_BF16) *reinterpret_cast<uint2*>(static_cast<uint16_t*>(p.out) + at) = make_uint2(f32_to_bf16x2_bits(out[0], out[1]), f32_to_bf16x2_bits(out[2], out[3]));
        else if (p.n % 4 == 0 && p.out_dtype == VIOLA_F16)
            *reinterpret_cast<uint2*>(static_cast<uint16_t*>(p.out) + at) = make_uint2(narrow16<f16_t>(out[0]) | narrow16<f16_t>(out[1]) << 16, narrow16<f16_t>(out[2]) | narrow16<f16_t>(out[3]) << 16);
        else
            for (int r = 0; r < 4 && col + r < p.n; ++r) store_float(p.out, at + r, p.out_dtype, out[r]);
    }
}

template <int MT, int NT, typename T> static int launch_rows(const Int8Args& p, const FusedArgs& f, hipStream_t stream) {
    const int64_t tiles = (p.n + 16 * NT - 1) / (16 * NT), row_tiles = int8_row_tiles(p, 16 * MT), steps = (p.k + 127) / 128;
    if (row_tiles >= 65536) return VIOLA_ETOOLARGE;                          // (groups and 16 rows each at most: fewer)
    // wavefronts that share a tile: as many as give every SIMD four, at least a step each
    const int64_t real = p.offsets ? p.m / (16 * MT) + (p.groups < p.m ? p.groups : p.m) : row_tiles;       // about
    int ks = ROWS_WAVES;
    while (ks > 1 && (tiles * real * ks > 4096 || steps < ks)) ks /= 2;
    const int64_t blocks = (tiles + ROWS_WAVES / ks - 1) / (ROWS_WAVES / ks);
    const size_t lds = (size_t)ROWS_WAVES * MT * NT * WAVE * 16 + (std::is_same<T, void>::value ? 0 : (size_t)p.m * (steps * 128 + 16));
    VIOLA_LAUNCH((int8_rows<MT, NT, T>), dim3((unsigned)blocks, (unsigned)row_tiles), 64 * ROWS_WAVES, (unsigned)lds, stream, p, f, ks);
    return viola_launch_status();
}

// Where the tiles of int8_gemm.hip are worse: a tile of 128 x 128 takes 5.5 us for 1024 of k, whether its rows are there or not and however few the CUs that have one, while here
// each 16 or 32 rows read the weights again. us, here and there: 64 x 4096 -> 4096 15 and 22, 128 x 4096 -> 4096 26 and 24, 128 x 4096 -> 1024 9 and 23, 64 x 4096 -> 11008 29 and 24; of groups,
// 4 rows each of 64 4096 -> 2048 98 and 157, 16 each 158 and 166, 31 each of 128 2048 -> 1024 124 and 89. Four tiles of channels for a wavefront share the loads of x where
// there are wavefronts enough without them: 32 x 4096 -> 11008 19 and 23 us, 32 x 4096 -> 4096 17 and 11.
bool int8_rows_fit(const Int8Args& p) { return p.offsets ? p.m <= 16 * (int64_t)p.groups : p.m <= 32 || (p.m <= 512 && p.m * p.n <= 393216); }
int launch_int8_rows(const Int8Args& p, hipStream_t stream) {
    const FusedArgs none = {};
    if (p.offsets || p.m <= 16) return launch_rows<1, 1, void>(p, none, stream);
    return p.n >= 8192 ? launch_rows<2, 4, void>(p, none, stream) : launch_rows<2, 1, void>(p, none, stream);
}

}  // namespace viola

using namespace viola;

extern "C" int viola_int8_rows_linear(const void* x, int64_t pitch, int dtype, int64_t m, int64_t k, int activation, const int8_t* b, int64_t ldb, const float* sb, int64_t n,
                                      const void* bias, int bias_dtype, void* out, int out_dtype, viola_stream_t stream_) {
    hipStream_t stream = viola_enter(stream_);
    VIOLA_CHECK_ARG(m >= 0 && n > 0 && k > 0 && n < (int64_t{1} << 31) && viola_is_float(dtype) && viola_is_float(out_dtype) && (!bias || viola_is_float(bias_dtype)) &&
                    activation <= VIOLA_RELU && pitch >= (activation >= 0 ? 2 : 1) * k && ldb >= k && ldb % 16 == 0);
    if (m == 0) return 0;
    if (!fused_fits(m, k) || ldb > (int64_t{1} << 22)) return VIOLA_EUNSUPPORTED;
    VIOLA_CHECK_ARG(x && b && sb && out && reinterpret_cast<uintptr_t>(b) % 16 == 0);
    Int8Args p = {};
    p.b = b; p.sb = sb; p.bias = bias; p.out = out; p.m = m; p.n = n; p.k = k; p.ldb = ldb; p.ldo = n; p.bias_dtype = bias_dtype; p.out_dtype = out_dtype;
    const FusedArgs f = {x, pitch, (int)m, (int)k, activation};
    if (dtype == VIOLA_F32) return launch_rows<1, 1, float>(p, f, stream);
    return dtype == VIOLA_BF16 ? launch_rows<1, 1, bf16_t>(p, f, stream) : launch_rows<1, 1, f16_t>(p, f, stream);
}
