// Shared by the products of 8-bit integers: int8_gemm.hip (tiles from LDS) and int8_rows.hip (few rows).
#pragma once
#include "common.hpp"

namespace viola {

// out[r, c] = (sum_k a[r, k] b[c, k]) sa[r] sb[c] + bias[c]; with offsets rows offsets[g] to offsets[g + 1] have the g-th b and sb, and rows from offsets[groups]
// on are zero. The sum is exact: |a| <= 127, |b| <= 128, k <= 2^17.
struct Int8Args {
    const int8_t* a; const int8_t* b;
    const float* sa; const float* sb;                                        // sb null: ones
    const void* bias; void* out;
    int64_t m, n, k;                                                         // k: a's columns, whole 16-byte pieces (zeros past the end)
    int64_t lda, ldb, ldo;                                                   // lda, ldb: bytes, multiples of 16
    const int* offsets; int groups; int64_t b_stride;                        // bytes from one b to the next
    int bias_dtype, out_dtype;
    int tiles_m, tiles_n;
    const void* z; int64_t z_pitch; int activation;                          // gated (int8_gemm.hip): out [m, 2 n] = the gradient of z = [g | u] from the product dh; z null: not
};

constexpr int64_t INT8_MOST_K = 1 << 17, INT8_MOST_GROUPS = 1024;

// A row's scale as it is applied: out = (sum * s) * sb, times lift, plus bias in one rounding. Of a row of values near the largest float sum * s would be infinite before a channel's
// scale makes it small again, so it is taken 2^64 smaller until then; of every other row lift is 1, and the last step a sum.
struct RowFactor {
    float s, lift;
    __device__ __forceinline__ explicit RowFactor(float sa) : s(sa > 0x1p60f ? sa * 0x1p-64f : sa), lift(sa > 0x1p60f ? 0x1p64f : 1.0f) {}
};

// The rows of group g of the groups' own, and of those behind the last one (g = groups). Offsets that a program made by hand are taken within the rows and in order: a
// product must stay inside its buffers whatever they hold.
__device__ __forceinline__ void int8_group_rows(const Int8Args& p, int g, int& from, int& to) {
    const int m = (int)p.m;
    from = g <= p.groups ? p.offsets[g] : m;
    to = g < p.groups ? p.offsets[g + 1] : m;
    from = from < 0 ? 0 : from < m ? from : m;
    to = to < from ? from : to < m ? to : m;
}
// All row tiles of `rows` rows (each group has whole tiles of its own, the rows behind them too). Every lane of a wavefront has to call it, and the next one.
__device__ __forceinline__ int int8_count_tiles(const Int8Args& p, int rows) {
    int tiles = 0;
    for (int g = threadIdx.x % WAVE; g <= p.groups; g += WAVE) {
        int from, to;
        int8_group_rows(p, g, from, to);
        tiles += (to - from + rows - 1) / rows;
    }
#pragma unroll
    for (int d = 1; d < WAVE; d *= 2) tiles += __shfl_xor(tiles, d, WAVE);
    return __builtin_amdgcn_readfirstlane(tiles);
}
// Row tile `index`: its group (groups: rows that are zero), and its rows [begin, end). False: there are not so many.
__device__ __forceinline__ bool int8_row_tile(const Int8Args& p, int64_t index, int rows, int& group, int64_t& begin, int64_t& end) {
    if (!p.offsets) {
        group = 0;
        begin = index * rows;
        end = begin + rows < p.m ? begin + rows : p.m;
        return begin < p.m;
    }
    const int lane = threadIdx.x % WAVE;
    int64_t before = 0;                                                      // tiles of the groups so far
    for (int base = 0; base <= p.groups; base += WAVE) {
        int from, to;
        int8_group_rows(p, base + lane, from, to);
        const int tiles = base + lane <= p.groups ? (to - from + rows - 1) / rows : 0;
        int upto = tiles;
#pragma unroll
        for (int d = 1; d < WAVE; d *= 2) {
            const int other = __shfl_up(upto, d, WAVE);
            upto += lane >= d ? other : 0;
        }
        const int64_t want = index - before;
        const uint64_t past = __ballot((int64_t)upto > want);
        if (past) {
            const int at = __ffsll((long long)past) - 1;
            group = __builtin_amdgcn_readfirstlane(base + at);
            const int skipped = __builtin_amdgcn_readfirstlane(__shfl(upto - tiles, at, WAVE));
            const int first = __builtin_amdgcn_readfirstlane(__shfl(from, at, WAVE)), last = __builtin_amdgcn_readfirstlane(__shfl(to, at, WAVE));
            begin = first + (want - skipped) * rows;
            end = begin + rows < last ? begin + rows : last;
            return true;
        }
        before += __builtin_amdgcn_readfirstlane(__shfl(upto, WAVE - 1, WAVE));
    }
    return false;
}
// (tiles of rows that a launch has to provide for: each group can leave one unfilled)
inline int64_t int8_row_tiles(const Int8Args& p, int rows) { return (p.m + rows - 1) / rows + (p.offsets ? p.groups + 1 : 0); }

// Whether the rows are few enough for int8_rows.hip, and the product there
bool int8_rows_fit(const Int8Args& p);
int launch_int8_rows(const Int8Args& p, hipStream_t stream);

}  // namespace viola
