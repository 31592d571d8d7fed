// Rows of floats as rows of 8-bit integers: what int8.hip does for whole tensors and int8_rows.hip on the way into a product.
#pragma once
#include "block_ops.hpp"

namespace viola {

// Eight values of a row from column c on; zero past the end.
template <typename T> __device__ __forceinline__ void load8(const T* row, int c, int cols, bool whole, bool stream, float (&v)[8]) {
    if (whole && c + 8 <= cols) {
        if constexpr (sizeof(T) == 4) {
            const uint4 a = stream ? load16<true>(reinterpret_cast<const uint4*>(row + c)) : load16<false>(reinterpret_cast<const uint4*>(row + c));
            const uint4 b = stream ? load16<true>(reinterpret_cast<const uint4*>(row + c + 4)) : load16<false>(reinterpret_cast<const uint4*>(row + c + 4));
            v[0] = __uint_as_float(a.x); v[1] = __uint_as_float(a.y); v[2] = __uint_as_float(a.z); v[3] = __uint_as_float(a.w);
            v[4] = __uint_as_float(b.x); v[5] = __uint_as_float(b.y); v[6] = __uint_as_float(b.z); v[7] = __uint_as_float(b.w);
        } else {
            const uint4 a = stream ? load16<true>(reinterpret_cast<const uint4*>(row + c)) : load16<false>(reinterpret_cast<const uint4*>(row + c));
            const uint32_t words[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                v[2 * i] = widen16<T>(words[i] & 0xffffu);
                v[2 * i + 1] = widen16<T>(words[i] >> 16);
            }
        }
        return;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = c + i < cols ? to_f32<T>(row[c + i]) : 0.0f;
}

__device__ __forceinline__ uint32_t magnitudes(const float (&v)[8], uint32_t most) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const uint32_t m = __float_as_uint(v[i]) & 0x7fffffffu;              // as integers: a NaN is above Inf, which is above all numbers
        most = m > most ? m : most;
    }
    return most;
}

// The scale of a row whose largest magnitude has these bits, and what its values are multiplied by.
struct RowScale {
    float s, lifted, inverse, lift;                                          // lifted = s lift, a normal number: tiny rows are quantized 2^64 larger
    __device__ __forceinline__ explicit RowScale(uint32_t most) {
        const float amax = __uint_as_float(most);
        const bool finite = most < 0x7f800000u;
        s = finite ? amax / 127.0f : __uint_as_float(0x7fc00000u);
        lift = amax < 0x1p-60f ? 0x1p64f : 1.0f;
        lifted = s * lift;
        inverse = finite && s > 0.0f ? 1.0f / lifted : 0.0f;
    }
};

// Eight values -> eight codes. Adding 1.5 2^23 rounds to an integer, whose low byte is the code.
__device__ __forceinline__ uint2 encode8_int(const float (&v)[8], const RowScale& r) {
    constexpr float MAGIC = 12582912.0f;
    uint32_t word[8];
    float far = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float t = v[i] * r.inverse, b = t + MAGIC;
        word[i] = __float_as_uint(b);
        far = fmaxf(far, fabsf(t - (b - MAGIC)));
    }
    // (the rare row that is lifted takes the exact way too, where codes are cut off at 127)
    if (far > 0.4998f || r.lift != 1.0f) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float x = v[i] * r.lift, half = 0.5f * r.lifted;
            float q = rintf(x * r.inverse);
            const float e = fmaf(-q, r.lifted, x);
            const bool odd = (int)q & 1;
            if (e > half || (e == half && odd)) q += 1.0f;
            else if (e < -half || (e == -half && odd)) q -= 1.0f;
            q = r.inverse == 0.0f ? 0.0f : __builtin_amdgcn_fmed3f(q, -127.0f, 127.0f);
            word[i] = (uint32_t)(int)q;
        }
    }
    if (r.inverse == 0.0f) return make_uint2(0, 0);                          // zeros, or a row that holds an Inf or a NaN
    auto pack = [](uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
        return __builtin_amdgcn_perm(__builtin_amdgcn_perm(d, c, 0x0c0c0400u), __builtin_amdgcn_perm(b, a, 0x0c0c0400u), 0x05040100u);
    };
    return make_uint2(pack(word[0], word[1], word[2], word[3]), pack(word[4], word[5], word[6], word[7]));
}

}  // namespace viola
