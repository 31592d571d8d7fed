// Rows of tokens to the experts and back. positions[t, j] is the row of token t's j-th expert (negative: none); the rows in use are
// the first `total` ones, which the router numbered without a gap.
//
//   scatter   rows[positions[t, j]] = gates[t, j] x[t]       (dispatch with gates of one, the gradient of gather's rows)
//   gather    out[t] = sum_j gates[t, j] rows[positions[t, j]]                                    (combine, dispatch's gradient)
//   and beside the second use of scatter the gates' gradient, dgates[t, j] = sum_c dout[t, c] rows[positions[t, j], c].
//
// Both are bound by memory: every row is read or written once, and a token's own row once for all of its experts.
#include "block_ops.hpp"

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
};

// one wavefront for each token; four tokens in a block
template <typename T> __global__ __launch_bounds__(256) void gather_kernel(RowsArgs a) {
    const int lane = threadIdx.x % 64;
    for (int64_t t = (int64_t)blockIdx.x * 4 + threadIdx.x / 64; t < a.tokens; t += (int64_t)gridDim.x * 4) {
        const int* at = a.positions + t * a.top_k;
        for (int c = lane; c < a.cols; c += 64) {
            float sum = 0.0f;
            for (int j = 0; j < a.top_k; ++j) {
                const int row = at[j];
                if (row < 0 || row >= a.rows) continue;
                const float v = to_f32<T>(static_cast<const T*>(a.in)[row * a.pitch + c]);
                sum = a.gates ? fmaf(a.gates[t * a.top_k + j], v, sum) : sum + v;
            }
            static_cast<T*>(a.out)[t * a.cols + c] = from_f32<T>(sum);
        }
    }
}

template <typename T> __global__ __launch_bounds__(256) void scatter_kernel(RowsArgs a) {
    const int lane = threadIdx.x % 64;
    T* out = static_cast<T*>(a.out);
    for (int64_t t = (int64_t)blockIdx.x * 4 + threadIdx.x / 64; t < a.tokens; t += (int64_t)gridDim.x * 4) {
        const T* x = static_cast<const T*>(a.in) + t * a.pitch;
        for (int j = 0; j < a.top_k; ++j) {
            const int row = a.positions[t * a.top_k + j];
            const bool there = row >= 0 && row < a.rows;
            float dot = 0.0f;
            if (there) {
                const float gate = a.gates ? a.gates[t * a.top_k + j] : 1.0f;
                for (int c = lane; c < a.cols; c += 64) {
                    const float v = to_f32<T>(x[c]);
                    if (out) out[(int64_t)row * a.cols + c] = a.gates ? from_f32<T>(gate * v) : x[c];
                    if (a.dots) dot = fmaf(v, to_f32<T>(static_cast<const T*>(a.values)[row * a.values_pitch + c]), dot);
                }
            }
            if (a.dots) {
                dot = wave_total(dot);
                if (lane == 0) a.dots[t * a.top_k + j] = dot;
            }
        }
        // rows that no token has
        if (out && a.total)
            for (int64_t row = (*a.total > 0 ? *a.total : 0) + t; row < a.rows; row += a.tokens)
                for (int c = lane; c < a.cols; c += 64) out[row * a.cols + c] = from_f32<T>(0.0f);
    }
}

int check(const RowsArgs& a, int dtype) {
    VIOLA_CHECK_ARG(viola_is_float(dtype) && a.tokens >= 0 && a.rows >= 0 && a.top_k > 0 && a.cols > 0);
    VIOLA_CHECK_ARG(a.tokens < (1LL << 31) && a.tokens * a.top_k < (1LL << 31) && a.rows < (1LL << 31));
    return 0;
}

unsigned blocks_for(int64_t tokens) { return (unsigned)((tokens + 3) / 4 < 1 << 20 ? (tokens + 3) / 4 : 1 << 20); }

}  // namespace

extern "C" int viola_rows_gather(const void* rows, int64_t pitch, int64_t row_count, int dtype, int64_t cols, const int32_t* positions, const float* gates, int64_t tokens,
                                 int top_k, void* out, viola_stream_t stream_) {
    hipStream_t stream = viola_enter(stream_);
    VIOLA_CHECK_ARG(cols > 0 && cols < (1LL << 31));
    RowsArgs a = {positions, gates, nullptr, tokens, row_count, pitch, top_k, (int)cols, rows, nullptr, 0, out, nullptr};
    if (const int status = check(a, dtype)) return status;
    if (tokens == 0) return 0;
    VIOLA_CHECK_ARG(positions && out && (rows || row_count == 0) && pitch >= cols);
    const unsigned grid = blocks_for(tokens);
    if (dtype == VIOLA_BF16) VIOLA_LAUNCH(gather_kernel<bf16_t>, grid, 256, 0, stream, a);
    else if (dtype == VIOLA_F16) VIOLA_LAUNCH(gather_kernel<f16_t>, grid, 256, 0, stream, a);
    else VIOLA_LAUNCH(gather_kernel<float>, grid, 256, 0, stream, a);
    return viola_launch_status();
}

extern "C" int viola_rows_scatter(const void* x, int64_t pitch, int dtype, int64_t cols, const int32_t* positions, const float* gates, int64_t tokens, int top_k,
                                  const int32_t* total, void* rows, int64_t row_count, const void* values, int64_t values_pitch, float* dots, viola_stream_t stream_) {
    hipStream_t stream = viola_enter(stream_);
    VIOLA_CHECK_ARG(cols > 0 && cols < (1LL << 31));
    RowsArgs a = {positions, gates, total, tokens, row_count, pitch, top_k, (int)cols, x, values, values_pitch, rows, dots};
    if (const int status = check(a, dtype)) return status;
    if (tokens == 0) return 0;
    VIOLA_CHECK_ARG(positions && x && pitch >= cols && (rows || dots || row_count == 0) && (!dots || values || row_count == 0) && (!dots || values_pitch >= cols));
    const unsigned grid = blocks_for(tokens);
    if (dtype == VIOLA_BF16) VIOLA_LAUNCH(scatter_kernel<bf16_t>, grid, 256, 0, stream, a);
    else if (dtype == VIOLA_F16) VIOLA_LAUNCH(scatter_kernel<f16_t>, grid, 256, 0, stream, a);
    else VIOLA_LAUNCH(scatter_kernel<float>, grid, 256, 0, stream, a);
    return viola_launch_status();
}
