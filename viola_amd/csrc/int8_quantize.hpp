// Rows of floats as rows of 8-bit integers: what int8.hip does for whole tensors and int8_rows.hip on the way into a product.
#pragma once
#include "block_ops.hpp"

namespace viola {

// 16 bytes at any address that a value may have: one load all the same, which the hardware cuts at cache lines
typedef uint32_t loose4 __attribute__((ext_vector_type(4), aligned(2)));
__device__ __forceinline__ uint4 load16_at(const void* from) {
    const loose4 w = *static_cast<const loose4*>(from);
    return make_uint4(w.x, w.y, w.z, w.w);
}

// Eight values of a row from column c on, as they are stored; zero past the end. Apart from their conversion, so that loads can be under way while other work goes on.
template <typename T> struct Raw8 {
    uint4 word[sizeof(T) / 2];
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (size_t i = 0; i < sizeof(T) / 2; ++i) word[i] = make_uint4(0, 0, 0, 0);
    }
    __device__ __forceinline__ void load(const T* row, int c, int cols) {
        if (c + 8 <= cols) {
#pragma unroll
            for (size_t i = 0; i < sizeof(T) / 2; ++i) word[i] = load16_at(row + c + 4 * i);
            return;
        }
        uint32_t w[2 * sizeof(T)];
#pragma unroll
        for (int i = 0; i < (int)(2 * sizeof(T)); ++i) w[i] = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            if (c + i >= cols) continue;
            if constexpr (sizeof(T) == 4) w[i] = __float_as_uint(row[c + i]);
            else w[i / 2] |= (uint32_t)reinterpret_cast<const uint16_t*>(row)[c + i] << (i % 2 * 16);
        }
#pragma unroll
        for (size_t i = 0; i < sizeof(T) / 2; ++i) word[i] = make_uint4(w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]);
    }
    __device__ __forceinline__ void widen(float (&v)[8]) const {
#pragma unroll
        for (size_t i = 0; i < sizeof(T) / 2; ++i) {
            const uint32_t w[4] = {word[i].x, word[i].y, word[i].z, word[i].w};
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                if constexpr (sizeof(T) == 4) {
                    v[4 * i + e] = __uint_as_float(w[e]);
                } else {
                    v[2 * e] = widen16<T>(w[e] & 0xffffu);
                    v[2 * e + 1] = widen16<T>(w[e] >> 16);
                }
            }
        }
    }
};
template <typename T> __device__ __forceinline__ void load8(const T* row, int c, int cols, float (&v)[8]) {
    Raw8<T> raw;
    raw.load(row, c, cols);
    raw.widen(v);
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
        const float b = fmaf(v[i], r.inverse, MAGIC);
        word[i] = __float_as_uint(b);
        far = fmaxf(far, fabsf(fmaf(v[i], r.inverse, MAGIC - b)));
    }
    // (the rare row that is lifted takes the exact way too, where codes are cut off at 127)
    if (far > 0.49998f || r.lift != 1.0f) {
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
