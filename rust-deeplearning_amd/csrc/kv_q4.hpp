// kv_q4.hpp -- the 4-bit cache's blocks on the device (RDL_KV_Q4,
// include/rdl_attention.h): 32 values of one position and head as a scale d
// and codes n, value = d (n - 8).  d has 8 significant bits and n - 8 at most
// 3, so a value is an f16 number without a rounding: the attention's products
// are those of an f16 cache.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "rdl_device.hpp"

namespace rdl {

constexpr int Q4_BLOCK = 32;
constexpr float Q4_MOST = 8160.0f;         // largest scale: 8 times it lies within f16
constexpr uint32_t Q4_NAN = 0x7E00u;       // the scale of a block with a value that is not finite
// A head's page: the codes of its positions, then their scales.
__host__ __device__ __forceinline__ int64_t q4_run_bytes(int64_t positions, int hd) {
    return positions * (hd / 2 + hd / Q4_BLOCK * 2);
}
__device__ __forceinline__ int q4_scale_at(int positions, int hd, int pos, int dim) {
    return positions * (hd / 2) + (pos * (hd / Q4_BLOCK) + dim / Q4_BLOCK) * 2;
}

typedef _Float16 q4h2 __attribute__((ext_vector_type(2)));

// From codes to values.  A nibble under an exponent is a whole number of steps above a power of two:
// 1024 + n in bits 0 .. 3 of f16, 64 + n in bits 4 .. 7.  The constants are kept from
// the compiler, so that they are registers and v_and_or_b32 takes both at once.
struct Q4Decoder {
    uint32_t low = 0x000F000Fu, high = 0x00F000F0u, from1024 = 0x64006400u, from64 = 0x54005400u;
    __device__ __forceinline__ Q4Decoder() {
        asm("" : "+s"(low), "+s"(high), "+v"(from1024), "+v"(from64));
    }
    // nibble t of both halves of x, times d
    __device__ __forceinline__ uint32_t pair(uint32_t x, int t, q4h2 d) const {
        const uint32_t y = t & 2 ? x >> 8 : x;
        const q4h2 n = __builtin_bit_cast(q4h2, t & 1 ? (y & high) | from64 : (y & low) | from1024);
        const _Float16 bias = t & 1 ? (_Float16)72.0f : (_Float16)1032.0f;
        return __builtin_bit_cast(uint32_t, (n - q4h2{bias, bias}) * d);
    }
    // the 8 values of a code word, in order
    __device__ __forceinline__ u32x4 word(uint32_t w, q4h2 d) const { return {pair(w, 0, d), pair(w, 1, d), pair(w, 2, d), pair(w, 3, d)}; }
};

// The scale of a block: mag, the bits of its largest magnitude, and whether a
// positive value, or a zero of either sign, has it.  f16 bits.
__device__ __forceinline__ uint32_t q4_scale(uint32_t mag, bool positive) {
    if (mag >= 0x7F800000u) return Q4_NAN;
    const uint32_t u = __builtin_bit_cast(uint32_t, as_f32((int32_t)mag) * 0.125f);
    const uint32_t b = (u + 0x7FFFu + (u >> 16 & 1)) & 0xFFFF0000u;  // 8 significant bits, to nearest
    const _Float16 h = (_Float16)fminf(as_f32((int32_t)b), Q4_MOST);
    return (uint32_t)__builtin_bit_cast(uint16_t, h) | (positive ? 0x8000u : 0u);
}
// What a block's values are divided by: its scale as f32, or 1 where that is 0 (its values, below 2^-21 all of
// them, then have code 8; 1 / 0 would make NaN of their quotients).
__device__ __forceinline__ float q4_divisor(uint32_t scale) {
    const float d = h2f(scale);
    return d == 0.0f ? 1.0f : d;
}
// The code of x under divisor d (inv: 1 / d or so): x / d to the nearest
// whole number, halves to even, which the rounded quotient alone would miss
// beside a half: the remainder of the nearest code, exact in f32, decides.
// HALF: x is an f16 number, 2^-14 of itself or more away from the halves that it is not: the quotient rounded
// to f32 has the same nearest whole number.
template <bool HALF = false>
__device__ __forceinline__ uint32_t q4_code(float x, float d, float inv) {
    if constexpr (HALF) {
        const float q = x * inv;
        return (uint32_t)(int)(fminf(fmaxf(rintf(fmaf(fmaf(-q, d, x), inv, q)), -8.0f), 7.0f) + 8.0f);
    }
    float c = rintf(x * inv);
    const float rest = fmaf(-c, d, x), twice = 2.0f * fabsf(rest), size = fabsf(d);
    const float step = (__builtin_bit_cast(uint32_t, rest) ^ __builtin_bit_cast(uint32_t, d)) >> 31 ? -1.0f : 1.0f;
    const bool odd = ((int)c & 1) != 0;  // (far out, where the code is cut, either will do)
    if (twice > size || (twice == size && odd)) c += step;
    return (uint32_t)(int)(fminf(fmaxf(c, -8.0f), 7.0f) + 8.0f);
}

}  // namespace rdl
