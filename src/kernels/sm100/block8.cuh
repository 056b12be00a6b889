// Activations in 8 bits: a block of neighbouring elements shares a power of two.
//
// With a = floor(log2 max|x|) over the block, the step is 2^q, q = max(a - 6, low), and an element is kept as its sign and
// m = min(rint(|x| / 2^q), 127), so x^ = +-m 2^q. The step is a power of two so that the division, the product and x^ itself are
// exact in the input's own type (m has 7 bits; bf16 holds 8, and low keeps 2^q a normal number of fp32 and bf16, of fp16 its
// smallest subnormal): a kept value is the same number wherever it is read, in matrix products too. |x^ - x| <= 2^(q-1), for the few
// elements above 127.5 steps 2^q: at most 2^-6 of the block's largest magnitude, 2^-7 where nothing is clamped.
//
// A code is sign << 7 | m and not two's complement because 0x4300 | m is the bf16 number 128 + m: a code widens without a
// conversion instruction. The scale byte is q + 127, so that it is the exponent field of the step; 255 marks a block that held an
// infinity or NaN: its codes are 0 and 0 * inf = NaN, so that every gradient made from the block says so.
#pragma once

#include "kernels/sm100/vec.cuh"

namespace b200ccl::dev {

constexpr unsigned kBlock8 = 32;  // elements of a block of an activation's row

template <typename T>
constexpr unsigned kLowScale8 = 1u;  // -126 + 127
template <>
constexpr unsigned kLowScale8<__half> = 103u;  // -24 + 127

// `amax`: the largest magnitude as bits of an fp32 number without sign, whose order is that of unsigned integers with infinities
// and NaN at the top.
template <typename T>
__device__ __forceinline__ unsigned scale8(unsigned amax) {
    const int e = (int)(amax >> 23) - 6;
    return e > 248 ? 255u : (unsigned)max(e, (int)kLowScale8<T>);
}
// 2^-q, what an element is multiplied with; 0 for a block that is not finite.
__device__ __forceinline__ float inverse_step8(unsigned scale) { return __uint_as_float(scale == 255u ? 0u : (254u - scale) << 23); }
__device__ __forceinline__ float step8(unsigned scale) { return __uint_as_float(scale << 23); }

// Adding 2^23 rounds to the nearest whole number, ties to even; the product before it is exact inside the fma.
__device__ __forceinline__ unsigned encode8(float x, float inverse) {
    const unsigned m = __float_as_uint(fmaf(fabsf(x), inverse, 8388608.0f)) & 0xffu;
    return min(m, 127u) | (__float_as_uint(x) >> 24 & 0x80u);
}
// Byte i of `word` as a number.
template <int i>
__device__ __forceinline__ float decode8(unsigned word, float step) {
    const unsigned m = __byte_perm(word & 0x7f7f7f7fu, 0x4b000000u, 0x7440 | i);  // 2^23 + m
    const float v = (__uint_as_float(m) - 8388608.0f) * step;
    return __uint_as_float(__float_as_uint(v) | (word << (24 - 8 * i) & 0x80000000u));
}
__device__ __forceinline__ void decode8x4(unsigned word, float step, float* f) {
    f[0] = decode8<0>(word, step);
    f[1] = decode8<1>(word, step);
    f[2] = decode8<2>(word, step);
    f[3] = decode8<3>(word, step);
}
__device__ __forceinline__ unsigned encode8x4(const float* f, float inverse) {
    return encode8(f[0], inverse) | encode8(f[1], inverse) << 8 | encode8(f[2], inverse) << 16 | encode8(f[3], inverse) << 24;
}
// A block that is not finite: x * 0 would be NaN, whose low bits are anything.
__device__ __forceinline__ unsigned finite8(unsigned word, unsigned scale) { return scale == 255u ? 0u : word; }

__device__ __forceinline__ unsigned magnitude_bits(float x) { return __float_as_uint(x) & 0x7fffffffu; }

}  // namespace b200ccl::dev
