// Rows of tokens to the experts and back. positions[t, j] is the row of token t's j-th expert (negative: none); the rows in use are
// the first `total` ones, which the router numbered without a gap.
//
//   scatter   rows[positions[t, j]] = gates[t, j] x[t]       (dispatch with gates of one, the gradient of gather's rows)
//   gather    out[t] = sum_j gates[t, j] rows[positions[t, j]]                                    (combine, dispatch's gradient)
//   and beside the second use of scatter the gates' gradient, dgates[t, j] = sum_c dout[t, c] rows[positions[t, j], c].
//
// Both are bound by memory: every row is read or written once, and a token's own row once for all of its experts.
#include "block_ops.hpp"

#include <type_traits>

using namespace viola;

namespace {

struct RowsArgs {
    const int* positions;
    const float* gates;                                                      // null: ones
    const int* total;                                                        // rows in use, on the device; null: all are
    int64_t tokens, rows, pitch;                                             // pitch: of the tokens (scatter), of the rows (gather)
    int top_k, cols;
    const void* in;
    const void* values;                                                      // scatter with dots: the rows themselves
    int64_t values_pitch;
    void* out;
    float* dots;
    bool stream_in, stream_out;                                              // rows are read, written past the caches' order
};

// ---------------------------------------------------------------------------------------------------- any width and address
// Where the rows are no whole 16-byte pieces. A wavefront for each token, which takes its rows by columns: f(first, number) for a lane's columns first,
// first + 64, ..: APART at a time as far as all lanes have them, then two, then one, so that accesses are of neighbours and several are under way.
// 16384 rows of 1001 in bf16, two choices: dispatch 33 us, sum 27, combine 27, its gradient 54 (one at a time: 42, 71, 81 and 83); 2.9 to 3.7 TB/s, where
// whole pieces reach 4.8 to 6: an access of two bytes a lane is an eighth of what a load can carry.
constexpr int APART = 8;
template <typename F> __device__ __forceinline__ void by_columns(int cols, F&& f) {
    const int lane = threadIdx.x % 64;
    int c = 0;
    for (; c + 64 * APART <= cols; c += 64 * APART) f(c + lane, std::integral_constant<int, APART>());
    for (; c + 64 * 2 <= cols; c += 64 * 2) f(c + lane, std::integral_constant<int, 2>());
    for (c += lane; c < cols; c += 64) f(c, std::integral_constant<int, 1>());
}

// A wavefront's pieces of work, `waves` in all: one, or beyond MOST_BLOCKS blocks several.
constexpr int64_t MOST_BLOCKS = 1 << 22;
template <typename F> __device__ __forceinline__ void each_wave(int64_t waves, F&& f) {
    for (int64_t wave = (int64_t)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x / 64); wave < waves; wave += (int64_t)gridDim.x * 4) f(wave);
}
unsigned blocks_for(int64_t waves) { return (unsigned)((waves + 3) / 4 < MOST_BLOCKS ? (waves + 3) / 4 : MOST_BLOCKS); }

template <typename T> __global__ __launch_bounds__(256) void gather_any_kernel(RowsArgs a) {
    each_wave(a.tokens, [&](int64_t t) {
        by_columns(a.cols, [&](int first, auto number) {
            constexpr int N = decltype(number)::value;
            float sum[N] = {};
            for (int j = 0; j < a.top_k; ++j) {
                const int row = a.positions[t * a.top_k + j];
                if (row < 0 || row >= a.rows) continue;
                const float gate = a.gates ? a.gates[t * a.top_k + j] : 1.0f;
                const T* from = static_cast<const T*>(a.in) + row * a.pitch + first;
                T v[N];
#pragma unroll
                for (int i = 0; i < N; ++i) v[i] = from[64 * i];
#pragma unroll
                for (int i = 0; i < N; ++i) sum[i] = fmaf(gate, to_f32<T>(v[i]), sum[i]);
            }
            T* to = static_cast<T*>(a.out) + t * a.cols + first;
#pragma unroll
            for (int i = 0; i < N; ++i) to[64 * i] = from_f32<T>(sum[i]);
        });
    });
}

template <typename T> __global__ __launch_bounds__(256) void scatter_any_kernel(RowsArgs a) {
    T* out = static_cast<T*>(a.out);
    each_wave(a.tokens, [&](int64_t t) {
        const T* x = static_cast<const T*>(a.in) + t * a.pitch;
        for (int j = 0; j < a.top_k; ++j) {
            const int row = a.positions[t * a.top_k + j];
            const bool there = row >= 0 && row < a.rows;
            float dot = 0.0f;
            if (there) {
                const float gate = a.gates ? a.gates[t * a.top_k + j] : 1.0f;
                by_columns(a.cols, [&](int first, auto number) {
                    constexpr int N = decltype(number)::value;
                    T v[N], u[N];
#pragma unroll
                    for (int i = 0; i < N; ++i) v[i] = x[first + 64 * i];
                    if (a.dots) {
                        const T* value = static_cast<const T*>(a.values) + row * a.values_pitch + first;
#pragma unroll
                        for (int i = 0; i < N; ++i) u[i] = value[64 * i];
#pragma unroll
                        for (int i = 0; i < N; ++i) dot = fmaf(to_f32<T>(v[i]), to_f32<T>(u[i]), dot);
                    }
                    if (!out) return;
                    T* to = out + (int64_t)row * a.cols + first;
                    if (a.gates) {
#pragma unroll
                        for (int i = 0; i < N; ++i) v[i] = from_f32<T>(gate * to_f32<T>(v[i]));
                    }
#pragma unroll
                    for (int i = 0; i < N; ++i) to[64 * i] = v[i];
                });
            }
            if (a.dots) {
                dot = wave_total(dot);
                if (threadIdx.x % 64 == 0) a.dots[t * a.top_k + j] = dot;
            }
        }
        // rows that no token has
        if (out && a.total)
            for (int64_t row = (*a.total > 0 ? *a.total : 0) + t; row < a.rows; row += a.tokens)
                for (int c = threadIdx.x % 64; c < a.cols; c += 64) out[row * a.cols + c] = from_f32<T>(0.0f);
    });
}

// ---------------------------------------------------------------------------------------------------- rows of whole 16-byte pieces
// A wavefront takes PIECES pieces a lane of one token's row and the same ones of its experts' rows, CHOICES of them at a time. Which token and which
// rows is the same for all lanes, so addresses are a scalar's work, and CHOICES * PIECES loads are in flight before the first is used: four to eight of them, which is
// what its launches choose by top_k. Rows of up to 64 pieces take one piece a lane, as more would leave lanes without work.
// At a large copy's rate: 16384 tokens of 4096 in bf16 to two experts 58 us (6.9 TB/s, part of it in the memory-side cache), the sum back 67 us (6.0); 16384 tokens of
// 1024 from eight experts 54 us (5.6), their gradients 114 us (5.0, rows and dots in one pass: each row of the experts read and written once).
template <typename T> constexpr int WIDE = 16 / sizeof(T);                   // elements of a piece

template <typename T> __device__ __forceinline__ void widen(const uint4& p, float (&v)[WIDE<T>]) {
    const uint32_t w[4] = {p.x, p.y, p.z, p.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if constexpr (sizeof(T) == 4) {
            v[i] = __uint_as_float(w[i]);
        } else {
            v[2 * i] = widen16<T>(w[i] & 0xffffu);
            v[2 * i + 1] = widen16<T>(w[i] >> 16);
        }
    }
}
template <typename T> __device__ __forceinline__ uint4 narrow(const float (&v)[WIDE<T>]) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if constexpr (sizeof(T) == 4) w[i] = __float_as_uint(v[i]);
        else if constexpr (__is_same(T, bf16_t)) w[i] = f32_to_bf16x2_bits(v[2 * i], v[2 * i + 1]);
        else w[i] = narrow16<T>(v[2 * i]) | narrow16<T>(v[2 * i + 1]) << 16;
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
}

// The row of a choice, 0 with `there` false for none: the load of an absent row is that of row 0, and its values are not used.
__device__ __forceinline__ int row_of(const RowsArgs& a, int64_t token, int j, bool& there) {
    const int row = j < a.top_k ? a.positions[token * a.top_k + j] : -1;
    there = row >= 0 && row < a.rows;
    return there ? row : 0;
}

template <typename T, int CHOICES, int PIECES> __global__ __launch_bounds__(256) void gather_kernel(RowsArgs a) {
    const int width = a.cols / WIDE<T>, cuts = (width + 64 * PIECES - 1) / (64 * PIECES);
    each_wave(a.tokens * cuts, [&](int64_t wave) {
        const int64_t token = wave / cuts;
        const int first = (int)(wave % cuts) * 64 * PIECES + threadIdx.x % 64;
        float sum[PIECES][WIDE<T>] = {};
        for (int j0 = 0; j0 < a.top_k; j0 += CHOICES) {
            uint4 piece[CHOICES][PIECES];
            const uint4* from[CHOICES];
            bool there[CHOICES];
#pragma unroll
            for (int j = 0; j < CHOICES; ++j) from[j] = reinterpret_cast<const uint4*>(static_cast<const T*>(a.in) + row_of(a, token, j0 + j, there[j]) * a.pitch);
            auto load = [&](auto stream) {
#pragma unroll
                for (int j = 0; j < CHOICES; ++j) {
#pragma unroll
                    for (int p = 0; p < PIECES; ++p) piece[j][p] = load16<decltype(stream)::value>(from[j] + (first + 64 * p < width ? first + 64 * p : 0));
                }
            };
            a.stream_in ? load(std::true_type()) : load(std::false_type());
#pragma unroll
            for (int j = 0; j < CHOICES; ++j) {
                if (!there[j]) continue;
                const float gate = a.gates ? a.gates[token * a.top_k + j0 + j] : 1.0f;
#pragma unroll
                for (int p = 0; p < PIECES; ++p) {
                    float v[WIDE<T>];
                    widen<T>(piece[j][p], v);
#pragma unroll
                    for (int i = 0; i < WIDE<T>; ++i) sum[p][i] = fmaf(gate, v[i], sum[p][i]);
                }
            }
        }
        uint4* to = reinterpret_cast<uint4*>(static_cast<T*>(a.out) + token * a.cols);
#pragma unroll
        for (int p = 0; p < PIECES; ++p)
            if (first + 64 * p < width) store16(to + first + 64 * p, narrow<T>(sum[p]), a.stream_out);
    });
}

template <typename T, int PIECES> __global__ __launch_bounds__(256) void scatter_kernel(RowsArgs a) {
    const int width = a.cols / WIDE<T>, cuts = (width + 64 * PIECES - 1) / (64 * PIECES);
    each_wave(a.tokens * cuts, [&](int64_t wave) {
        const int64_t token = wave / cuts;
        const int first = (int)(wave % cuts) * 64 * PIECES + threadIdx.x % 64;
        const uint4* from = reinterpret_cast<const uint4*>(static_cast<const T*>(a.in) + token * a.pitch);
        uint4 piece[PIECES];
#pragma unroll
        for (int p = 0; p < PIECES; ++p) piece[p] = from[first + 64 * p < width ? first + 64 * p : 0];
        for (int j = 0; j < a.top_k; ++j) {
            bool there;
            uint4* to = reinterpret_cast<uint4*>(static_cast<T*>(a.out) + (int64_t)row_of(a, token, j, there) * a.cols);
            if (!there) continue;
            const float gate = a.gates ? a.gates[token * a.top_k + j] : 1.0f;
#pragma unroll
            for (int p = 0; p < PIECES; ++p) {
                uint4 word = piece[p];
                if (a.gates) {
                    float v[WIDE<T>];
                    widen<T>(piece[p], v);
#pragma unroll
                    for (int i = 0; i < WIDE<T>; ++i) v[i] *= gate;
                    word = narrow<T>(v);
                }
                if (first + 64 * p < width) store16(to + first + 64 * p, word, a.stream_out);
            }
        }
        // rows that no token has
        if (a.total)
            for (int64_t row = (*a.total > 0 ? *a.total : 0) + token; row < a.rows; row += a.tokens) {
                uint4* to = reinterpret_cast<uint4*>(static_cast<T*>(a.out) + row * a.cols);
#pragma unroll
                for (int p = 0; p < PIECES; ++p)
                    if (first + 64 * p < width) to[first + 64 * p] = make_uint4(0, 0, 0, 0);
            }
    });
}

// scatter and the dots beside it: WAVES wavefronts to a token, which take its row in turn, PIECES pieces a lane at a time, so that a dot is summed in
// one place.
template <typename T, int CHOICES, int PIECES, int WAVES> __global__ __launch_bounds__(256) void scatter_dots_kernel(RowsArgs a) {
    __shared__ float parts[WAVES][CHOICES];
    const int width = a.cols / WIDE<T>, lane = threadIdx.x % 64;
    each_wave(a.tokens * WAVES, [&](int64_t wave) {                          // with several wavefronts a block is one token, and so all of it makes a turn
        const int64_t token = wave / WAVES;
        const int part = (int)(wave % WAVES);
        const uint4* from = reinterpret_cast<const uint4*>(static_cast<const T*>(a.in) + token * a.pitch);
        for (int j0 = 0; j0 < a.top_k; j0 += CHOICES) {
            const uint4* value[CHOICES];
            uint4* to[CHOICES];
            float gate[CHOICES], dot[CHOICES] = {};
            bool there[CHOICES];
#pragma unroll
            for (int j = 0; j < CHOICES; ++j) {
                const int64_t row = row_of(a, token, j0 + j, there[j]);
                value[j] = reinterpret_cast<const uint4*>(static_cast<const T*>(a.values) + row * a.values_pitch);
                to[j] = reinterpret_cast<uint4*>(static_cast<T*>(a.out) + row * a.cols);
                gate[j] = a.gates && there[j] ? a.gates[token * a.top_k + j0 + j] : 1.0f;
            }
            for (int first = part * 64 * PIECES + lane; first - lane < width; first += WAVES * 64 * PIECES) {
                uint4 piece[PIECES], other[CHOICES][PIECES];
                auto load = [&](auto stream) {
#pragma unroll
                    for (int p = 0; p < PIECES; ++p) {
                        const int c = first + 64 * p < width ? first + 64 * p : 0;
                        piece[p] = load16<decltype(stream)::value>(from + c);
#pragma unroll
                        for (int j = 0; j < CHOICES; ++j) other[j][p] = load16<decltype(stream)::value>(value[j] + c);
                    }
                };
                a.stream_in ? load(std::true_type()) : load(std::false_type());
#pragma unroll
                for (int p = 0; p < PIECES; ++p) {
                    const bool in = first + 64 * p < width;
                    float v[WIDE<T>];
                    widen<T>(piece[p], v);
#pragma unroll
                    for (int j = 0; j < CHOICES; ++j) {
                        if (!there[j]) continue;
                        float u[WIDE<T>], sum = 0.0f;
                        widen<T>(other[j][p], u);
#pragma unroll
                        for (int i = 0; i < WIDE<T>; ++i) {
                            sum = fmaf(v[i], u[i], sum);
                            u[i] = gate[j] * v[i];
                        }
                        if (in) {
                            dot[j] += sum;
                            if (a.out) store16(to[j] + first + 64 * p, a.gates ? narrow<T>(u) : piece[p], a.stream_out);
                        }
                    }
                }
            }
#pragma unroll
            for (int j = 0; j < CHOICES; ++j) {
                dot[j] = wave_total(dot[j]);
                if constexpr (WAVES == 1) {
                    if (lane == 0 && j0 + j < a.top_k) a.dots[token * a.top_k + j0 + j] = dot[j];
                } else if (lane == 0) {
                    parts[part][j] = dot[j];
                }
            }
            if constexpr (WAVES > 1) {
                __syncthreads();
                if ((int)threadIdx.x < CHOICES && j0 + (int)threadIdx.x < a.top_k) {
                    float sum = 0.0f;
#pragma unroll
                    for (int w = 0; w < WAVES; ++w) sum += parts[w][threadIdx.x];
                    a.dots[token * a.top_k + j0 + threadIdx.x] = sum;
                }
                __syncthreads();
            }
        }
        if (a.out && a.total)
            for (int64_t row = (*a.total > 0 ? *a.total : 0) + token; row < a.rows; row += a.tokens) {
                uint4* to = reinterpret_cast<uint4*>(static_cast<T*>(a.out) + row * a.cols);
                for (int c = part * 64 + lane; c < width; c += WAVES * 64) to[c] = make_uint4(0, 0, 0, 0);
            }
    });
}

// ---------------------------------------------------------------------------------------------------- launches
bool whole_pieces(const RowsArgs& a, int dtype) {
    const int size = viola_dtype_size(dtype);
    for (const void* p : {a.in, a.values, (const void*)a.out})
        if (reinterpret_cast<uintptr_t>(p) % 16) return false;
    return a.cols * (int64_t)size % 16 == 0 && a.pitch * size % 16 == 0 && (!a.dots || a.values_pitch * size % 16 == 0) && a.rows > 0;
}

template <typename T, int CHOICES, int PIECES> void launch_gather(const RowsArgs& a, hipStream_t stream) {
    const int64_t cuts = (a.cols / WIDE<T> + 64 * PIECES - 1) / (64 * PIECES);
    VIOLA_LAUNCH((gather_kernel<T, CHOICES, PIECES>), blocks_for(a.tokens * cuts), 256, 0, stream, a);
}
template <typename T, int PIECES> void launch_scatter(const RowsArgs& a, hipStream_t stream) {
    const int64_t cuts = (a.cols / WIDE<T> + 64 * PIECES - 1) / (64 * PIECES);
    VIOLA_LAUNCH((scatter_kernel<T, PIECES>), blocks_for(a.tokens * cuts), 256, 0, stream, a);
}
template <typename T, int CHOICES, int PIECES> void launch_dots(const RowsArgs& a, hipStream_t stream) {
    // Four wavefronts to a token where its row has a piece for every lane of them (16384 tokens of 4096 in BF16, two choices: 130 against 155 us with one
    // wavefront), one below (1024, eight choices: 112 against 125 us).
    const int64_t width = a.cols / WIDE<T>;
    if (width <= 64) VIOLA_LAUNCH((scatter_dots_kernel<T, CHOICES, 1, 1>), blocks_for(a.tokens), 256, 0, stream, a);
    else if (width < 256) VIOLA_LAUNCH((scatter_dots_kernel<T, CHOICES, PIECES, 1>), blocks_for(a.tokens), 256, 0, stream, a);
    else VIOLA_LAUNCH((scatter_dots_kernel<T, CHOICES, 1, 4>), blocks_for(a.tokens * 4), 256, 0, stream, a);
}

template <typename T> void run_gather(const RowsArgs& a, int dtype, hipStream_t stream) {
    const bool narrow_rows = a.cols / WIDE<T> <= 64;
    if (!whole_pieces(a, dtype)) VIOLA_LAUNCH(gather_any_kernel<T>, blocks_for(a.tokens), 256, 0, stream, a);
    else if (a.top_k == 1) narrow_rows ? launch_gather<T, 1, 1>(a, stream) : launch_gather<T, 1, 4>(a, stream);
    else if (a.top_k == 2) narrow_rows ? launch_gather<T, 2, 1>(a, stream) : launch_gather<T, 2, 2>(a, stream);
    else if (a.top_k <= 4) launch_gather<T, 4, 1>(a, stream);
    else launch_gather<T, 8, 1>(a, stream);
}

template <typename T> void run_scatter(const RowsArgs& a, int dtype, hipStream_t stream) {
    if (!whole_pieces(a, dtype)) VIOLA_LAUNCH(scatter_any_kernel<T>, blocks_for(a.tokens), 256, 0, stream, a);
    else if (!a.dots) a.cols / WIDE<T> <= 64 ? launch_scatter<T, 1>(a, stream) : launch_scatter<T, 2>(a, stream);
    else if (a.top_k == 1) launch_dots<T, 1, 4>(a, stream);
    else if (a.top_k == 2) launch_dots<T, 2, 4>(a, stream);
    else if (a.top_k <= 4) launch_dots<T, 4, 2>(a, stream);
    else launch_dots<T, 8, 1>(a, stream);
}

int check(const RowsArgs& a, int dtype) {
    VIOLA_CHECK_ARG(viola_is_float(dtype) && a.tokens >= 0 && a.rows >= 0 && a.top_k > 0 && a.cols > 0);
    VIOLA_CHECK_ARG(a.tokens < (1LL << 31) && a.tokens * a.top_k < (1LL << 31) && a.rows < (1LL << 31));
    return 0;
}

}  // namespace

extern "C" int viola_rows_gather(const void* rows, int64_t pitch, int64_t row_count, int dtype, int64_t cols, const int32_t* positions, const float* gates, int64_t tokens,
                                 int top_k, void* out, viola_stream_t stream_) {
    hipStream_t stream = viola_enter(stream_);
    VIOLA_CHECK_ARG(cols > 0 && cols <= 1 << 28);
    RowsArgs a = {positions, gates, nullptr, tokens, row_count, pitch, top_k, (int)cols, rows, nullptr, 0, out, nullptr};
    if (const int status = check(a, dtype)) return status;
    if (tokens == 0) return 0;
    a.stream_in = tokens * top_k * cols * viola_dtype_size(dtype) > STREAM_IN;
    a.stream_out = tokens * cols * viola_dtype_size(dtype) > STREAM_OUT;
    VIOLA_CHECK_ARG(positions && out && (rows || row_count == 0) && pitch >= cols);
    if (dtype == VIOLA_BF16) run_gather<bf16_t>(a, dtype, stream);
    else if (dtype == VIOLA_F16) run_gather<f16_t>(a, dtype, stream);
    else run_gather<float>(a, dtype, stream);
    return viola_launch_status();
}

extern "C" int viola_rows_scatter(const void* x, int64_t pitch, int dtype, int64_t cols, const int32_t* positions, const float* gates, int64_t tokens, int top_k,
                                  const int32_t* total, void* rows, int64_t row_count, const void* values, int64_t values_pitch, float* dots, viola_stream_t stream_) {
    hipStream_t stream = viola_enter(stream_);
    VIOLA_CHECK_ARG(cols > 0 && cols <= 1 << 28);
    RowsArgs a = {positions, gates, total, tokens, row_count, pitch, top_k, (int)cols, x, values, values_pitch, rows, dots};
    if (const int status = check(a, dtype)) return status;
    if (tokens == 0) return 0;
    a.stream_in = dots && tokens * top_k * cols * viola_dtype_size(dtype) > STREAM_IN;
    a.stream_out = rows && row_count * cols * viola_dtype_size(dtype) > STREAM_OUT;
    VIOLA_CHECK_ARG(positions && x && pitch >= cols && (rows || dots || row_count == 0) && (!dots || values || row_count == 0) && (!dots || values_pitch >= cols));
    if (dtype == VIOLA_BF16) run_scatter<bf16_t>(a, dtype, stream);
    else if (dtype == VIOLA_F16) run_scatter<f16_t>(a, dtype, stream);
    else run_scatter<float>(a, dtype, stream);
    return viola_launch_status();
}
