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

// 16 bytes that are not looked at again soon. Stores past the caches' order (a call that writes more than STREAM_OUT) leave room there for what
// is: 16384 rows of 1152 in BF16 through norm_between take 32 instead of 40 us. Loads likewise, where a call reads more than the memory-side
// cache holds anyway (STREAM_IN): 268 MB of rows through combine 5.3 instead of 4.9 TB/s; what fits there is faster left to it (a tenth of that: 8.7 against 6.9 us).
constexpr int64_t STREAM_OUT = 4 << 20, STREAM_IN = 128 << 20;
typedef uint32_t words4 __attribute__((ext_vector_type(4)));
// The empty statements keep the two kinds apart: the compiler makes one access, of the plain kind, of two alternatives that differ in the hint only.
template <bool STREAM> __device__ __forceinline__ uint4 load16(const uint4* from) {
    if constexpr (!STREAM) return *from;
    asm volatile("");
    const words4 w = __builtin_nontemporal_load(reinterpret_cast<const words4*>(from));
    asm volatile("");
    return make_uint4(w.x, w.y, w.z, w.w);
}
__device__ __forceinline__ void store16(uint4* to, const uint4& v, bool stream) {
    if (stream) {
        asm volatile("");
        __builtin_nontemporal_store(words4{v.x, v.y, v.z, v.w}, reinterpret_cast<words4*>(to));
        asm volatile("");
    } else {
        *to = v;
    }
}

}  // namespace viola
