// Helpers shared by the kernels around a block (norm.hip, rows.hip, route.hip): sums over a wavefront on the vector ALU, and sums
// over the wavefronts of a block.
#pragma once

#include "common.hpp"

namespace viola {

template <int CTRL> __device__ __forceinline__ float dpp_add(float v) {
    return v + __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, 0xf, 0xf, true));
}

// The sum over the 64 lanes, in every lane. DPP moves only (no LDS crossbar): xor 1, xor 2, halves of eight and of sixteen
// mirrored (their halves hold equal sums by then), then lane 15 and lane 31 broadcast into the rows behind them; lane 63 has the
// whole sum. The order is the same on every call.
__device__ __forceinline__ float wave_total(float v) {
    v = dpp_add<0xB1>(v);                                                    // quad_perm 1 0 3 2
    v = dpp_add<0x4E>(v);                                                    // quad_perm 2 3 0 1
    v = dpp_add<0x141>(v);                                                   // row_half_mirror
    v = dpp_add<0x140>(v);                                                   // row_mirror
    v += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x142, 0xa, 0xf, true));   // row_bcast:15 into rows 1 and 3
    v += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x143, 0xc, 0xf, true));   // row_bcast:31 into rows 2 and 3
    return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), 63));
}

// Sums over all threads of a block of at most 16 wavefronts, in every thread. Two sets of slots are used in turn, so one barrier a
// sum is enough: a wavefront writes a set again only behind the barrier of the sum in between, which all others reach after
// they have read it. Every thread of the block has to call it.
struct BlockSums {
    float2 (*slot)[16];                                                      // two sets in LDS
    int waves, wave, turn = 0;
    __device__ __forceinline__ BlockSums(float2 (*slots)[16]) : slot(slots), waves((blockDim.x + 63) / 64), wave(threadIdx.x / 64) {}
    __device__ __forceinline__ float2 both(float a, float b) {
        a = wave_total(a);
        b = wave_total(b);
        if (waves == 1) return make_float2(a, b);
        if (threadIdx.x % 64 == 0) slot[turn][wave] = make_float2(a, b);
        __syncthreads();
        float2 sum = slot[turn][0];
        for (int w = 1; w < waves; ++w) {
            sum.x += slot[turn][w].x;
            sum.y += slot[turn][w].y;
        }
        turn ^= 1;
        return sum;
    }
    __device__ __forceinline__ float one(float a) {
        a = wave_total(a);
        if (waves == 1) return a;
        if (threadIdx.x % 64 == 0) slot[turn][wave].x = a;
        __syncthreads();
        float sum = slot[turn][0].x;
        for (int w = 1; w < waves; ++w) sum += slot[turn][w].x;
        turn ^= 1;
        return sum;
    }
};

}  // namespace viola
