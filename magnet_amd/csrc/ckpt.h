// Encoding of the 8-bit activation checkpoints (the format is described in ckpt.hip).
#pragma once
#include <cstdint>

#include <hip/hip_runtime.h>

namespace mhckpt {

constexpr int kBlockCols = 32;

// the largest magnitude of four values as float bits: an unsigned maximum orders them, non-finite values on top
__device__ inline uint32_t magnitude(float4 v) {
    const uint32_t x = __float_as_uint(v.x) & 0x7fffffffu, y = __float_as_uint(v.y) & 0x7fffffffu;
    const uint32_t z = __float_as_uint(v.z) & 0x7fffffffu, w = __float_as_uint(v.w) & 0x7fffffffu;
    const uint32_t a = x > y ? x : y, b = z > w ? z : w;
    return a > b ? a : b;
}

// scale byte s + 128 of a block whose largest magnitude has these bits: exponent field E means p = E - 126, so s = E - 133,
// one more from 127.5 / 128 of the next power of two on
__device__ inline uint32_t scale_byte(uint32_t top) {
    if (top >= 0x7f800000u) return 0u;
    int s = int(top >> 23) - 133 + ((top & 0x7fffffu) >= 0x7f0000u ? 1 : 0);
    s = s < -110 ? -110 : s > 121 ? 121 : s;
    return uint32_t(s + 128);
}

// 2^s of a scale byte: the exponent field is s + 127.  The byte 0 of a block that is not finite gives -inf, which its zero codes
// turn into NaN; the byte 1, which no block has, gives 0.
__device__ inline float scale_of(uint32_t e) { return __uint_as_float((e - 1u) << 23); }

__device__ inline uint32_t encode1(float x, float inverse) {
    float q = rintf(x * inverse);
    q = fminf(fmaxf(q, -127.0f), 127.0f);
    return uint32_t(int(q) + 128);
}

__device__ inline uint32_t encode(float4 v, uint32_t e) {
    // 1 / 2^s has the exponent field 127 - (e - 128) = 255 - e, between 6 and 237; a block that is not finite keeps no codes
    const float inverse = __uint_as_float((255u - e) << 23);
    if (e == 0u) return 0x80808080u;
    return encode1(v.x, inverse) | (encode1(v.y, inverse) << 8) | (encode1(v.z, inverse) << 16) | (encode1(v.w, inverse) << 24);
}

// (u - 128) 2^s, both steps exact
__device__ inline float decode1(uint32_t u, float s) { return (float(u) - 128.0f) * s; }
__device__ inline float4 decode(uint32_t code, uint32_t e) {
    const float s = scale_of(e);
    return make_float4(decode1(code & 255u, s), decode1((code >> 8) & 255u, s), decode1((code >> 16) & 255u, s), decode1(code >> 24, s));
}

}  // namespace mhckpt
