// Norms before and after a block with its gate and residual sum (norm.hpp), and the gradients of the vectors along the row.
#include "norm_launch.hpp"

#include <initializer_list>

using namespace viola;

// norm_rows_*.hip
#define VIOLA_NORM_ROWS(TX, TY)                                                                             \
    extern template void viola::norm_forward_rows<TX, TY>(const NormArgs&, int, dim3, hipStream_t);         \
    extern template void viola::norm_backward_rows<TX, TY>(const NormArgs&, int, bool, bool, dim3, hipStream_t);
VIOLA_NORM_ROWS(bf16_t, bf16_t)
VIOLA_NORM_ROWS(f16_t, f16_t)
VIOLA_NORM_ROWS(float, float)
VIOLA_NORM_ROWS(float, bf16_t)
VIOLA_NORM_ROWS(float, f16_t)
VIOLA_NORM_ROWS(loose_t, loose_t)

namespace {

// ---------------------------------------------------------------------------------------------------- rows too wide for a block's registers
// Beyond ROW_COLUMNS, of any type and address: a block for each row at a time, element by element; what a row needs twice is read again, from cache.
// Columns stay with their thread, so sums over the rows of a portion can be kept in the portion's own slots. Narrower rows, odd ones too, are faster in
// registers: between two blocks, forward and backward, 178 and 942 us here against 86 and 184 there for 64 x 256 rows of 1001 in bf16.
struct Columns {
    const NormArgs& a;
    int64_t row, group;
    float4 stat;                                                             // mu_y, r_y, mu_x, r_x as far as they are known
    __device__ __forceinline__ float vector(const void* data, int64_t at, int dtype, int c, float absent) const { return data ? load_float(data, at + c, dtype) : absent; }
    __device__ __forceinline__ float y_hat(int c) const { return (load_float(a.y, row * a.y_pitch + c, a.branch_dtype) - stat.x) * stat.y; }
    __device__ __forceinline__ float gate(int c) const { return a.alpha * vector(a.gate.data, group * a.gate.pitch, a.vector_dtype, c, 1.0f); }
    __device__ __forceinline__ float after_weight(int c) const { return vector(a.after_weight, 0, a.weight_dtype, c, 1.0f); }
    __device__ __forceinline__ float out(int c) const {
        const float x = load_float(a.x, row * a.x_pitch + c, a.x_dtype);
        if (!a.y) return x;
        return fmaf(a.rho, x, gate(c) * fmaf(y_hat(c), after_weight(c), vector(a.after_bias, 0, a.weight_dtype, c, 0.0f)));
    }
    __device__ __forceinline__ float scale(int c) const { return 1.0f + vector(a.scale.data, group * a.scale.pitch, a.vector_dtype, c, 0.0f); }
    __device__ __forceinline__ float weight(int c) const { return vector(a.weight, 0, a.weight_dtype, c, 1.0f); }
};

// mu and r of a row given by its columns. The mean first and the deviations from it after that: a row far from zero keeps its digits.
template <typename F> __device__ __forceinline__ float2 statistics(const NormArgs& a, int kind, BlockSums& sums, F&& value) {
    float mean = 0.0f, s = 0.0f;
    if (kind == VIOLA_NORM_LAYER) {
        for (int c = threadIdx.x; c < a.cols; c += blockDim.x) s += value(c);
        mean = sums.one(s) / (float)a.cols;
    }
    s = 0.0f;
    for (int c = threadIdx.x; c < a.cols; c += blockDim.x) {
        const float d = value(c) - mean;
        s = fmaf(d, d, s);
    }
    return make_float2(mean, 1.0f / sqrtf(sums.one(s) / (float)a.cols + a.eps));
}

__global__ __launch_bounds__(256) void norm_forward_any_kernel(NormArgs a) {
    __shared__ float2 slots[2][16];
    BlockSums sums(slots);
    for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
        Columns at{a, row, row / a.group_rows, make_float4(0.0f, 1.0f, 0.0f, 1.0f)};
        if (a.y && a.after != VIOLA_NORM_NONE) {
            const float2 s = statistics(a, a.after, sums, [&](int c) { return load_float(a.y, row * a.y_pitch + c, a.branch_dtype); });
            at.stat.x = s.x;
            at.stat.y = s.y;
        }
        if (a.h) {
            const float2 s = statistics(a, a.before, sums, [&](int c) { return at.out(c); });
            at.stat.z = s.x;
            at.stat.w = s.y;
        }
        for (int c = threadIdx.x; c < a.cols; c += blockDim.x) {
            const float x = at.out(c);
            if (a.out) store_float(a.out, row * a.cols + c, a.x_dtype, x);
            if (a.h) {
                const float n = fmaf((x - at.stat.z) * at.stat.w, at.weight(c), at.vector(a.bias, 0, a.weight_dtype, c, 0.0f));
                store_float(a.h, row * a.cols + c, a.branch_dtype, fmaf(n, at.scale(c), at.vector(a.shift.data, at.group * a.shift.pitch, a.vector_dtype, c, 0.0f)));
            }
        }
        if (a.stats && threadIdx.x == 0) a.stats[row] = at.stat;
    }
}

// One portion: up to ceil(group_rows / per_group) rows of one group.
__global__ __launch_bounds__(256) void norm_backward_any_kernel(NormArgs a) {
    __shared__ float2 slots[2][16];
    BlockSums sums(slots);
    const float inverse = 1.0f / (float)a.cols;
    const int64_t length = (a.group_rows + a.per_group - 1) / a.per_group;
    const int count = __popc(a.sums);
    for (int64_t portion = blockIdx.x; portion < a.portions; portion += gridDim.x) {
        const int64_t group = portion / a.per_group, group_end = (group + 1) * a.group_rows;
        const int64_t begin = group * a.group_rows + portion % a.per_group * length;
        const int64_t end = begin + length < group_end ? begin + length : group_end;
        float* slot = a.parts + portion * count * a.cols;
        for (int c = threadIdx.x; c < a.cols; c += blockDim.x)
            for (int i = 0; i < count; ++i) slot[(int64_t)i * a.cols + c] = 0.0f;
        for (int64_t row = begin; row < end; ++row) {
            const Columns at{a, row, group, a.stats[row]};
            auto x_hat = [&](int c) { return (at.out(c) - at.stat.z) * at.stat.w; };
            auto dh = [&](int c) { return load_float(a.dh, row * a.cols + c, a.branch_dtype); };
            auto q = [&](int c) { return dh(c) * at.weight(c) * at.scale(c); };
            float m1 = 0.0f, m0 = 0.0f;
            if (a.dh) {
                float along = 0.0f, total = 0.0f;
                for (int c = threadIdx.x; c < a.cols; c += blockDim.x) {
                    along = fmaf(q(c), x_hat(c), along);
                    total += q(c);
                }
                const float2 both = sums.both(along, total);
                m1 = both.x * inverse;
                m0 = a.before == VIOLA_NORM_LAYER ? both.y * inverse : 0.0f;
            }
            auto d = [&](int c) {
                const float from_out = a.dout ? load_float(a.dout, row * a.cols + c, a.x_dtype) : 0.0f;
                return a.dh ? fmaf(at.stat.w, q(c) - fmaf(x_hat(c), m1, m0), from_out) : from_out;
            };
            float along = 0.0f, total = 0.0f;
            for (int c = threadIdx.x; c < a.cols; c += blockDim.x) {
                const float grad = d(c);
                if (a.dx) store_float(a.dx, row * a.cols + c, a.x_dtype, a.y ? a.rho * grad : grad);
                float* to = slot + c;
                if (a.y) {
                    const float hat = at.y_hat(c), p = grad * at.gate(c) * at.after_weight(c);
                    if (a.sums & SUM_A1) { *to = fmaf(grad, hat, *to); to += a.cols; }
                    if (a.sums & SUM_A0) { *to += grad; to += a.cols; }
                    along = fmaf(p, hat, along);
                    total += p;
                }
                if (a.dh) {
                    if (a.sums & SUM_S1) { *to = fmaf(dh(c), x_hat(c), *to); to += a.cols; }
                    if (a.sums & SUM_S0) *to += dh(c);
                }
            }
            if (!a.dy) continue;
            float n1 = 0.0f, n0 = 0.0f;
            if (a.after != VIOLA_NORM_NONE) {
                const float2 both = sums.both(along, total);
                n1 = both.x * inverse;
                n0 = a.after == VIOLA_NORM_LAYER ? both.y * inverse : 0.0f;
            }
            for (int c = threadIdx.x; c < a.cols; c += blockDim.x) {
                const float p = d(c) * at.gate(c) * at.after_weight(c);
                store_float(a.dy, row * a.cols + c, a.branch_dtype, a.after == VIOLA_NORM_NONE ? p : at.stat.y * (p - fmaf(at.y_hat(c), n1, n0)));
            }
        }
    }
}

// ---------------------------------------------------------------------------------------------------- sums over rows
struct ReduceArgs {
    const float* parts;
    int64_t portions, per_group;
    int cols, sums, weight_dtype, vector_dtype;
    float alpha;
    const void *after_weight, *after_bias, *weight, *bias;
    NormVector gate, scale;
    // one for all rows (vectors with a pitch of 0 too), or one for each group
    void *d_after_weight, *d_after_bias, *d_weight, *d_bias, *d_gate, *d_scale, *d_shift;
    int gate_by_group, scale_by_group, shift_by_group;
    int whole;                                                               // sections for gradients summed over all rows: 1 or 0
};

struct Sums { float a1, a0, s1, s0; };

constexpr int64_t MOST_SECTIONS = 32768;                                     // of groups: a grid has up to 65535 in y

// The wanted sums of one portion; `at`: where in the portion each lies.
struct PortionLayout {
    int sums, a0, s1, s0;
    int64_t stride;
    __device__ __forceinline__ PortionLayout(const ReduceArgs& a)
        : sums(a.sums), a0(__popc(a.sums & SUM_A1) * a.cols), s1(__popc(a.sums & (SUM_A1 | SUM_A0)) * a.cols), s0(__popc(a.sums & (SUM_A1 | SUM_A0 | SUM_S1)) * a.cols),
          stride((int64_t)__popc(a.sums) * a.cols) {}
    __device__ __forceinline__ Sums load(const float* from) const {
        Sums v = {0.0f, 0.0f, 0.0f, 0.0f};
        if (sums & SUM_A1) v.a1 = from[0];
        if (sums & SUM_A0) v.a0 = from[a0];
        if (sums & SUM_S1) v.s1 = from[s1];
        if (sums & SUM_S0) v.s0 = from[s0];
        return v;
    }
};

// Sections of blocks (blockIdx.y). `whole` of them, 1 or 0: what is summed over all rows, WIDTH columns by as many contiguous slices of the portions as 1024
// threads have, the slices then added in order. The others: what is summed group by group, WIDTH columns by a group for each slice.
template <int WIDTH> __global__ __launch_bounds__(1024) void norm_reduce_kernel(ReduceArgs a) {
    constexpr int SLICES = 1024 / WIDTH;
    __shared__ float piece[SLICES][8][WIDTH + 1];
    constexpr int TOGETHER = 4;                                              // portions whose loads are under way together
    const int c = threadIdx.x % WIDTH, slice = threadIdx.x / WIDTH, col = blockIdx.x * WIDTH + c;
    const PortionLayout layout(a);
    const bool in = col < a.cols;
    auto vector = [&](const void* data, int64_t at, int dtype, float absent) { return data && in ? load_float(data, at + col, dtype) : absent; };
    if ((int)blockIdx.y >= a.whole) {
        const int64_t group = (int64_t)(blockIdx.y - a.whole) * SLICES + slice;
        if (!in || group >= a.portions / a.per_group) return;
        float a1 = 0.0f, a0 = 0.0f, s1 = 0.0f, s0 = 0.0f;
        const float* from = a.parts + group * a.per_group * layout.stride + col;
#pragma unroll 4
        for (int64_t p = 0; p < a.per_group; ++p) {
            const Sums v = layout.load(from + p * layout.stride);
            a1 += v.a1; a0 += v.a0; s1 += v.s1; s0 += v.s0;
        }
        const int64_t to = group * a.cols + col;
        const float w_a = vector(a.after_weight, 0, a.weight_dtype, 1.0f), b_a = vector(a.after_bias, 0, a.weight_dtype, 0.0f);
        const float w_b = vector(a.weight, 0, a.weight_dtype, 1.0f), b_b = vector(a.bias, 0, a.weight_dtype, 0.0f);
        if (a.d_gate && a.gate_by_group) store_float(a.d_gate, to, a.vector_dtype, a.alpha * fmaf(w_a, a1, a.after_bias ? b_a * a0 : 0.0f));
        if (a.d_scale && a.scale_by_group) store_float(a.d_scale, to, a.vector_dtype, fmaf(w_b, s1, a.bias ? b_b * s0 : 0.0f));
        if (a.d_shift && a.shift_by_group) store_float(a.d_shift, to, a.vector_dtype, s0);
        return;
    }
    // the four sums, then the same under the gate and under one plus the scale
    float sum[8] = {};
    if (in) {
        const int64_t per = (a.portions + SLICES - 1) / SLICES;
        const int64_t begin = slice * per, end = begin + per < a.portions ? begin + per : a.portions;
        const bool gates = a.gate.pitch != 0, scales = a.scale.pitch != 0;   // one for each group: loaded with each portion
        const float all_g = vector(a.gate.data, 0, a.vector_dtype, 1.0f), all_s = 1.0f + vector(a.scale.data, 0, a.vector_dtype, 0.0f);
        auto gate_of = [&](int64_t p) { return gates ? vector(a.gate.data, (uint32_t)p / (uint32_t)a.per_group * a.gate.pitch, a.vector_dtype, 1.0f) : all_g; };
        auto scale_of = [&](int64_t p) { return scales ? 1.0f + vector(a.scale.data, (uint32_t)p / (uint32_t)a.per_group * a.scale.pitch, a.vector_dtype, 0.0f) : all_s; };
        auto add = [&](const Sums& v, float g, float s) {
            sum[0] += v.a1; sum[1] += v.a0; sum[2] += v.s1; sum[3] += v.s0;
            sum[4] = fmaf(g, v.a1, sum[4]); sum[5] = fmaf(g, v.a0, sum[5]); sum[6] = fmaf(s, v.s1, sum[6]); sum[7] = fmaf(s, v.s0, sum[7]);
        };
        const float* from = a.parts + begin * layout.stride + col;
        int64_t p = begin;
        for (; p + TOGETHER <= end; p += TOGETHER, from += TOGETHER * layout.stride) {
            Sums v[TOGETHER];
            float g[TOGETHER], s[TOGETHER];
#pragma unroll
            for (int u = 0; u < TOGETHER; ++u) {
                v[u] = layout.load(from + u * layout.stride);
                g[u] = gate_of(p + u);
                s[u] = scale_of(p + u);
            }
#pragma unroll
            for (int u = 0; u < TOGETHER; ++u) add(v[u], g[u], s[u]);
        }
        for (; p < end; ++p, from += layout.stride) add(layout.load(from), gate_of(p), scale_of(p));
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) piece[slice][i][c] = sum[i];
    __syncthreads();
    if (slice < 8) {
        float total = piece[0][slice][c];
#pragma unroll 8
        for (int u = 1; u < SLICES; ++u) total += piece[u][slice][c];
        piece[0][slice][c] = total;                                          // read by this thread only until the next barrier
    }
    __syncthreads();
    if (slice || !in) return;
    const float a1 = piece[0][0][c], a0 = piece[0][1][c], s1 = piece[0][2][c], s0 = piece[0][3][c];
    if (a.d_after_weight) store_float(a.d_after_weight, col, a.weight_dtype, a.alpha * piece[0][4][c]);
    if (a.d_after_bias) store_float(a.d_after_bias, col, a.weight_dtype, a.alpha * piece[0][5][c]);
    if (a.d_weight) store_float(a.d_weight, col, a.weight_dtype, piece[0][6][c]);
    if (a.d_bias) store_float(a.d_bias, col, a.weight_dtype, piece[0][7][c]);
    if (a.d_gate && !a.gate_by_group) {
        const float b_a = vector(a.after_bias, 0, a.weight_dtype, 0.0f);
        store_float(a.d_gate, col, a.vector_dtype, a.alpha * fmaf(vector(a.after_weight, 0, a.weight_dtype, 1.0f), a1, a.after_bias ? b_a * a0 : 0.0f));
    }
    if (a.d_scale && !a.scale_by_group) {
        const float b_b = vector(a.bias, 0, a.weight_dtype, 0.0f);
        store_float(a.d_scale, col, a.vector_dtype, fmaf(vector(a.weight, 0, a.weight_dtype, 1.0f), s1, a.bias ? b_b * s0 : 0.0f));
    }
    if (a.d_shift && !a.shift_by_group) store_float(a.d_shift, col, a.vector_dtype, s0);
}

// Whether rows of this width are held in registers; then f(stream type, branch type): in pieces of eight elements where types, widths and addresses are of
// whole pieces, loose otherwise.
template <typename F> bool in_registers(NormArgs& a, std::initializer_list<const void*> tensors, F&& f) {
    if (a.cols > ROW_COLUMNS) return false;
    a.team = (a.cols + 511) / 512 * 64;
    bool whole = a.cols % 8 == 0 && a.x_pitch % 8 == 0 && (!a.y || a.y_pitch % 8 == 0);
    for (const void* p : tensors) whole = whole && reinterpret_cast<uintptr_t>(p) % 16 == 0;
    for (const void* p : {a.after_weight, a.after_bias, a.weight, a.bias, a.gate.data, a.scale.data, a.shift.data}) whole = whole && reinterpret_cast<uintptr_t>(p) % 16 == 0;
    for (const NormVector& v : {a.gate, a.scale, a.shift}) whole = whole && v.pitch % 8 == 0;
    const int x = a.x_dtype, y = a.branch_dtype;
    if (whole && x == VIOLA_BF16 && y == VIOLA_BF16) f(bf16_t(), bf16_t());
    else if (whole && x == VIOLA_F16 && y == VIOLA_F16) f(f16_t(), f16_t());
    else if (whole && x == VIOLA_F32 && y == VIOLA_F32) f(float(), float());
    else if (whole && x == VIOLA_F32 && y == VIOLA_BF16) f(float(), bf16_t());
    else if (whole && x == VIOLA_F32 && y == VIOLA_F16) f(float(), f16_t());
    else f(loose_t(), loose_t());
    return true;
}
void stream(NormArgs& a, int64_t bytes_in, int64_t bytes_out) {
    a.stream_in = bytes_in > STREAM_IN;
    a.stream_out = bytes_out > STREAM_OUT;
}
bool plain(const NormArgs& a) { return a.after == VIOLA_NORM_NONE && !a.after_weight && !a.after_bias; }

// A portion for every block that the chip holds at once (16 wavefronts a CU), of two rows for each of its teams at least
// (2000 rows of 256: 14.7 us, with four 16.4) and of four (1024 rows of 4096: 20.3 us, with two 21.8), and of no more than one group.
int64_t portions_per_group(int64_t rows, int64_t group_rows, int64_t cols) {
    NormArgs a = {};
    a.team = (int)((cols + 511) / 512 * 64);
    const bool registers = cols <= ROW_COLUMNS;
    const int64_t block = registers ? norm_block(a, false) : 1024, teams = block / a.team, least = !registers ? 1 : teams > 1 ? 2 * teams : 4;
    const int64_t groups = rows / group_rows, wanted = (256 * (1024 / block) + groups - 1) / groups, most = (group_rows + least - 1) / least;
    return wanted < most ? wanted : most;
}

constexpr int64_t MOST_COLUMNS = 1 << 28;

bool valid_rows(const void* p, int64_t pitch, int64_t cols) { return p && pitch >= cols; }

int set_common(NormArgs& a, const void* x, int64_t x_pitch, int x_dtype, const void* y, int64_t y_pitch, int branch_dtype, int64_t rows, int64_t cols, int after,
               const void* after_weight, const void* after_bias, int before, const void* weight, const void* bias, int weight_dtype, const void* gate,
               int64_t gate_pitch, const void* scale, int64_t scale_pitch, const void* shift, int64_t shift_pitch, int vector_dtype, int64_t group_rows, float rho,
               float alpha, float eps) {
    VIOLA_CHECK_ARG(viola_is_float(x_dtype) && viola_is_float(branch_dtype) && viola_is_float(weight_dtype) && viola_is_float(vector_dtype));
    VIOLA_CHECK_ARG(rows >= 0 && cols > 0 && group_rows > 0 && rows % group_rows == 0);
    VIOLA_CHECK_ARG(after >= VIOLA_NORM_NONE && after <= VIOLA_NORM_LAYER && before >= VIOLA_NORM_NONE && before <= VIOLA_NORM_LAYER && eps >= 0.0f);
    for (int64_t pitch : {gate_pitch, scale_pitch, shift_pitch}) VIOLA_CHECK_ARG(pitch == 0 || pitch >= cols);
    VIOLA_CHECK_ARG(cols <= MOST_COLUMNS);
    a.x = x; a.y = y; a.x_pitch = x_pitch; a.y_pitch = y_pitch; a.rows = rows; a.group_rows = group_rows;
    a.cols = (int)cols; a.x_dtype = x_dtype; a.branch_dtype = branch_dtype; a.after = after; a.before = before;
    a.weight_dtype = weight_dtype; a.vector_dtype = vector_dtype;
    a.after_weight = after_weight; a.after_bias = after_bias; a.weight = weight; a.bias = bias;
    a.gate = {gate, gate_pitch}; a.scale = {scale, scale_pitch}; a.shift = {shift, shift_pitch};
    a.rho = rho; a.alpha = alpha; a.eps = eps;
    return 0;
}

}  // namespace

extern "C" int viola_norm_forward(const void* x, int64_t x_pitch, int x_dtype, const void* y, int64_t y_pitch, int branch_dtype, int64_t rows, int64_t cols, int after,
                                  const void* after_weight, const void* after_bias, int before, const void* weight, const void* bias, int weight_dtype,
                                  const void* gate, int64_t gate_pitch, const void* scale, int64_t scale_pitch, const void* shift, int64_t shift_pitch, int vector_dtype,
                                  int64_t group_rows, float residual_scale, float branch_scale, float eps, void* out, void* h, float* stats, viola_stream_t stream_) {
    hipStream_t hip_stream = viola_enter(stream_);
    NormArgs a = {};
    const int status = set_common(a, x, x_pitch, x_dtype, y, y_pitch, branch_dtype, rows, cols, after, after_weight, after_bias, before, weight, bias, weight_dtype, gate,
                                  gate_pitch, scale, scale_pitch, shift, shift_pitch, vector_dtype, group_rows, residual_scale, branch_scale, eps);
    if (status) return status;
    if (rows == 0) return 0;
    VIOLA_CHECK_ARG(valid_rows(x, x_pitch, cols) && (out || h) && (out != nullptr) == (y != nullptr) && (!y || y_pitch >= cols));
    VIOLA_CHECK_ARG((h != nullptr) == (before != VIOLA_NORM_NONE) && (reinterpret_cast<uintptr_t>(stats) % 16) == 0);
    const int form = !y ? FORM_BEFORE : !h ? FORM_AFTER : plain(a) ? FORM_PLAIN : FORM_BETWEEN;
    a.out = out; a.h = h; a.stats = reinterpret_cast<float4*>(stats);
    if (in_registers(a, {x, y, out, h}, [&](auto tx, auto ty) {
            // as many blocks as the chip holds at once by their registers: each loads the vectors along the row once
            const int64_t block = norm_block(a, true), teams = block / a.team, waves = form == FORM_BETWEEN ? 16 : 20, held = waves * 64 / block;
            const int64_t blocks = 256 * (held ? held : 1);
            a.chunk = ((rows + blocks - 1) / blocks + teams - 1) / teams * teams;
            stream(a, rows * cols * ((int)sizeof(tx) + (y ? (int)sizeof(ty) : 0)), rows * cols * ((out ? (int)sizeof(tx) : 0) + (h ? (int)sizeof(ty) : 0)));
            norm_forward_rows<decltype(tx), decltype(ty)>(a, form, dim3((unsigned)((rows + a.chunk - 1) / a.chunk)), hip_stream);
        }))
        return viola_launch_status();
    VIOLA_LAUNCH(norm_forward_any_kernel, dim3((unsigned)(rows < 65536 ? rows : 65536)), 256, 0, hip_stream, a);
    return viola_launch_status();
}

extern "C" int64_t viola_norm_portions(int64_t rows, int64_t cols, int64_t group_rows) {
    if (rows <= 0 || cols <= 0 || cols > MOST_COLUMNS || group_rows <= 0 || rows % group_rows) return 0;
    return rows / group_rows * portions_per_group(rows, group_rows, cols);
}

extern "C" int viola_norm_backward(const void* x, int64_t x_pitch, int x_dtype, const void* y, int64_t y_pitch, int branch_dtype, int64_t rows, int64_t cols, int after,
                                   const void* after_weight, const void* after_bias, int before, const void* weight, const void* bias, int weight_dtype,
                                   const void* gate, int64_t gate_pitch, const void* scale, int64_t scale_pitch, const void* shift, int64_t shift_pitch, int vector_dtype,
                                   int64_t group_rows, float residual_scale, float branch_scale, const float* stats, const void* dout, const void* dh, void* dx, void* dy,
                                   float* parts, int64_t parts_floats, void* d_after_weight, void* d_after_bias, void* d_weight, void* d_bias, void* d_gate,
                                   void* d_scale, void* d_shift, viola_stream_t stream_) {
    hipStream_t hip_stream = viola_enter(stream_);
    NormArgs a = {};
    const int status = set_common(a, x, x_pitch, x_dtype, y, y_pitch, branch_dtype, rows, cols, after, after_weight, after_bias, before, weight, bias, weight_dtype, gate,
                                  gate_pitch, scale, scale_pitch, shift, shift_pitch, vector_dtype, group_rows, residual_scale, branch_scale, 0.0f);
    if (status) return status;
    const bool gate_sums = d_gate && y, scale_sums = d_scale && dh;
    // rows of none: the sums over rows are still written, as zeros, by the reduction below
    if (rows) {
        VIOLA_CHECK_ARG((!dh || valid_rows(x, x_pitch, cols)) && stats && (!y || y_pitch >= cols) && (dh || y) && (dh != nullptr) == (before != VIOLA_NORM_NONE) && (y || !dy));
        VIOLA_CHECK_ARG(reinterpret_cast<uintptr_t>(stats) % 16 == 0);
    }
    a.stats = reinterpret_cast<float4*>(const_cast<float*>(stats));
    a.dout = dout; a.dh = dh; a.dx = dx; a.dy = dy; a.parts = parts;
    a.sums = (d_after_weight || gate_sums ? SUM_A1 : 0) | (d_after_bias || (gate_sums && after_bias) ? SUM_A0 : 0) | (d_weight || scale_sums ? SUM_S1 : 0) |
             (d_bias || d_shift || (scale_sums && bias) ? SUM_S0 : 0);
    a.per_group = rows ? portions_per_group(rows, group_rows, cols) : 1;
    a.portions = rows ? rows / group_rows * a.per_group : 0;
    if (a.sums && rows) VIOLA_CHECK_ARG(parts && parts_floats >= a.portions * __builtin_popcount((unsigned)a.sums) * cols);
    const bool grouped = (d_gate && gate_pitch) || (d_scale && scale_pitch) || (d_shift && shift_pitch);
    const bool whole = d_after_weight || d_after_bias || d_weight || d_bias || (d_gate && !gate_pitch) || (d_scale && !scale_pitch) || (d_shift && !shift_pitch);
    // Sums over all rows of few columns: 16 to a block, or there are too few blocks (50 x 197 rows of 768: 5.3 us, with 32 columns 6.6; 4096 columns 8.4 and 7.3).
    const bool narrow = whole && cols <= 1024;
    const int64_t width = narrow ? 16 : 32, slices = 1024 / width;
    const int64_t by_groups = grouped ? (rows / group_rows + slices - 1) / slices : 0;
    if (a.portions > UINT32_MAX) return VIOLA_EUNSUPPORTED;
    if (rows) {
        const dim3 grid((unsigned)(a.portions < 65536 ? a.portions : 65536));
        const int form = !y ? FORM_BEFORE : !dh ? FORM_AFTER : plain(a) ? FORM_PLAIN : FORM_BETWEEN;
        const bool with_bias = after_bias || (a.sums & SUM_A0), with_shift = (a.sums & SUM_S0) != 0;
        if (!in_registers(a, {x, y, dout, dh, dx, dy, parts}, [&](auto tx, auto ty) {
                const int64_t n = rows * cols, x_size = sizeof(tx), y_size = sizeof(ty);
                stream(a, n * ((dh ? x_size + y_size : 0) + (y ? y_size : 0) + (dout ? x_size : 0)), n * ((dx ? x_size : 0) + (dy ? y_size : 0)));
                norm_backward_rows<decltype(tx), decltype(ty)>(a, form, with_bias, with_shift, grid, hip_stream);
            }))
            VIOLA_LAUNCH(norm_backward_any_kernel, grid, 256, 0, hip_stream, a);
    }
    if (whole || by_groups) {
        ReduceArgs r = {};
        r.whole = whole;
        r.parts = parts; r.portions = a.portions; r.per_group = a.per_group; r.cols = (int)cols; r.sums = a.sums;
        r.weight_dtype = weight_dtype; r.vector_dtype = vector_dtype; r.alpha = branch_scale;
        r.after_weight = after_weight; r.after_bias = after_bias; r.weight = weight; r.bias = bias; r.gate = a.gate; r.scale = a.scale;
        r.d_after_weight = d_after_weight; r.d_after_bias = d_after_bias; r.d_weight = d_weight; r.d_bias = d_bias;
        r.d_gate = d_gate; r.d_scale = d_scale; r.d_shift = d_shift;
        r.gate_by_group = gate_pitch != 0; r.scale_by_group = scale_pitch != 0; r.shift_by_group = shift_pitch != 0;
        // A launch for every MOST_SECTIONS of groups: the next one's begin where this one's end.
        for (int64_t left = by_groups;;) {
            const int64_t sections = left < MOST_SECTIONS ? left : MOST_SECTIONS;
            const dim3 grid((unsigned)((cols + width - 1) / width), (unsigned)(r.whole + sections));
            if (narrow) VIOLA_LAUNCH(norm_reduce_kernel<16>, grid, 1024, 0, hip_stream, r);
            else VIOLA_LAUNCH(norm_reduce_kernel<32>, grid, 1024, 0, hip_stream, r);
            left -= sections;
            if (left <= 0) break;
            const int64_t groups = sections * slices;
            auto advance = [&](void*& p, int by_group) {
                if (p && by_group) p = static_cast<char*>(p) + groups * cols * viola_dtype_size(vector_dtype);
            };
            r.whole = 0;
            r.portions -= groups * a.per_group;
            r.parts += groups * a.per_group * __builtin_popcount((unsigned)a.sums) * cols;
            advance(r.d_gate, r.gate_by_group);
            advance(r.d_scale, r.scale_by_group);
            advance(r.d_shift, r.shift_by_group);
        }
    }
    return viola_launch_status();
}
