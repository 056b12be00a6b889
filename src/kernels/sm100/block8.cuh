// Activations in 8 bits: a block of neighbouring elements shares a power of two.
//
// With a = floor(log2 max|x|) over the block, the step is 2^q, q = max(a - 6, low), and an element is kept as its sign and
// m = min(rint(|x| / 2^q), 127), so x^ = +-m 2^q. The step is a power of two so that the division, the product and x^ itself are
// exact in the input's own type (m has 7 bits; bf16 holds 8, and low keeps 2^q a normal number of fp32 and bf16, of fp16 its
// smallest subnormal): a kept value is the same number wherever it is read, in matrix products too. |x^ - x| <= 2^(q-1), for the few
// elements above 127.5 steps 2^q: at most 2^-6 of the block's largest magnitude, 2^-7 where nothing is clamped.
//
// A code is sign << 7 | m and not two's complement, so that a code widens without a conversion instruction: as a bf16 number, sign << 15 | m is
// +-m 2^-133, exactly. And rounding needs none either: |x| 2^-q + 128 in bf16 (+ 1024 in fp16) is rounded to a whole number by its own
// last bit, ties to even. Both work on two elements at once. The scale byte is q + 127, so that it is the exponent field of the step; 255 marks a block that held an
// infinity or NaN: its codes are 0 and 0 * inf = NaN, so that every gradient made from the block says so.
#pragma once

#include "kernels/sm100/vec.cuh"

#include <type_traits>

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

// ---- 16-bit types, two elements in a word ----------------------------------------------------------------
__device__ __forceinline__ __nv_bfloat162 as_b2(unsigned w) { return *reinterpret_cast<__nv_bfloat162*>(&w); }
__device__ __forceinline__ __half2 as_h2(unsigned w) { return *reinterpret_cast<__half2*>(&w); }
__device__ __forceinline__ unsigned bits_of(__nv_bfloat162 v) { return *reinterpret_cast<unsigned*>(&v); }
__device__ __forceinline__ unsigned bits_of(__half2 v) { return *reinterpret_cast<unsigned*>(&v); }

// The larger magnitude of each half so far, NaN once there is one; and of both at the end, as fp32.
template <typename T>
__device__ __forceinline__ unsigned larger_magnitudes(unsigned so_far, unsigned word) {
    if constexpr (std::is_same_v<T, __half>) return bits_of(__hmax2_nan(as_h2(so_far), __habs2(as_h2(word))));
    else return bits_of(__hmax2_nan(as_b2(so_far), __habs2(as_b2(word))));
}
template <typename T>
__device__ __forceinline__ unsigned magnitude_of_pair(unsigned pair) {
    const unsigned m = max(pair & 0xffffu, pair >> 16);
    if constexpr (std::is_same_v<T, __half>) return __float_as_uint(__half2float(__ushort_as_half((unsigned short)m)));
    return m << 16;
}

// 2^-q for words of T: bf16 in one factor; fp16, which does not reach 2^24, in two.
template <typename T>
struct Inverse16 {
    unsigned a, b;
    __device__ __forceinline__ explicit Inverse16(unsigned scale) {
        if constexpr (std::is_same_v<T, __half>) {
            const int e = 127 - (int)scale, first = e >> 1, second = e - first;  // e from -9 to 24
            a = scale == 255u ? 0u : (unsigned)(15 + first) * 0x04000400u;
            b = scale == 255u ? 0u : (unsigned)(15 + second) * 0x04000400u;
        } else {
            a = scale == 255u ? 0u : (254u - scale) * 0x00800080u;
            b = 0u;
        }
    }
};
// Codes of the four elements of two words (of a block that is finite).
template <typename T>
__device__ __forceinline__ unsigned encode8x4(unsigned x, unsigned y, const Inverse16<T>& inverse) {
    unsigned mx, my;
    if constexpr (std::is_same_v<T, __half>) {
        const __half2 top = as_h2(0x647f647fu), magic = as_h2(0x64006400u);  // 1024 + 127, 1024
        mx = bits_of(__hmin2(__hfma2(__hmul2(__habs2(as_h2(x)), as_h2(inverse.a)), as_h2(inverse.b), magic), top));
        my = bits_of(__hmin2(__hfma2(__hmul2(__habs2(as_h2(y)), as_h2(inverse.a)), as_h2(inverse.b), magic), top));
    } else {
        const __nv_bfloat162 top = as_b2(0x437f437fu), magic = as_b2(0x43004300u);  // 128 + 127, 128
        mx = bits_of(__hmin2(__hfma2(__habs2(as_b2(x)), as_b2(inverse.a), magic), top));
        my = bits_of(__hmin2(__hfma2(__habs2(as_b2(y)), as_b2(inverse.a), magic), top));
    }
    return __byte_perm(mx, my, 0x6420) | (__byte_perm(x, y, 0x7531) & 0x80808080u);
}
// What widens codes to words of T. bf16: 2^(q + 6), behind a factor 2^127. fp16: 2^q.
template <typename T>
__device__ __forceinline__ unsigned step16(unsigned scale) {
    if constexpr (std::is_same_v<T, __half>) return bits_of(__float2half2_rn(step8(scale)));
    return min(scale + 6u, 255u) * 0x00800080u;
}
// Four codes as two words of T.
template <typename T>
__device__ __forceinline__ uint2 widen8x4(unsigned word, unsigned step) {
    const unsigned m = word & 0x7f7f7f7fu, sign = word & 0x80808080u;
    if constexpr (std::is_same_v<T, __half>) {
        // 1024 + m, less 1024, times the step: fp16 has no exponents left for the other way.
        const __half2 off = as_h2(0x64006400u);
        const unsigned a = bits_of(__hmul2(__hsub2(as_h2(__byte_perm(m, 0x64646464u, 0x4140)), off), as_h2(step)));
        const unsigned b = bits_of(__hmul2(__hsub2(as_h2(__byte_perm(m, 0x64646464u, 0x4342)), off), as_h2(step)));
        return make_uint2(a | __byte_perm(sign, 0u, 0x1404), b | __byte_perm(sign, 0u, 0x3424));
    } else {
        const __nv_bfloat162 far = as_b2(0x7f007f00u);  // 2^127
        return make_uint2(bits_of(__hmul2(__hmul2(as_b2(__byte_perm(m, sign, 0x5140)), far), as_b2(step))),
                          bits_of(__hmul2(__hmul2(as_b2(__byte_perm(m, sign, 0x7362)), far), as_b2(step))));
    }
}

__device__ __forceinline__ unsigned magnitude_bits(float x) { return __float_as_uint(x) & 0x7fffffffu; }

// N neighbouring elements at p, of which `count` are there; the others are zeros. p is a multiple of an element: the aligned 16 bytes that hold a wanted one
// are read, and shifted.
template <typename T, int N>
__device__ __forceinline__ void load_any(const char* p, unsigned count, unsigned (&w)[N * sizeof(T) / 4]) {
    constexpr unsigned W = N * sizeof(T) / 4, G = W / 4 + 1;
    const unsigned shift = (unsigned)(reinterpret_cast<std::uintptr_t>(p) & 15u);
    const char* base = p - shift;
    unsigned r[4 * G];
#pragma unroll
    for (unsigned g = 0; g < G; ++g) {
        const uint4 v = 16u * g < shift + count * (unsigned)sizeof(T) && count != 0u ? *reinterpret_cast<const uint4*>(base + 16 * g) : make_uint4(0u, 0u, 0u, 0u);
        r[4 * g] = v.x;
        r[4 * g + 1] = v.y;
        r[4 * g + 2] = v.z;
        r[4 * g + 3] = v.w;
    }
#pragma unroll
    for (unsigned i = 0; i < W + 2; ++i) r[i] = shift & 8u ? r[i + 2] : r[i];
#pragma unroll
    for (unsigned i = 0; i < W + 1; ++i) r[i] = shift & 4u ? r[i + 1] : r[i];
    if constexpr (sizeof(T) == 2) {
#pragma unroll
        for (unsigned i = 0; i < W; ++i) w[i] = shift & 2u ? __funnelshift_r(r[i], r[i + 1], 16) : r[i];
    } else {
#pragma unroll
        for (unsigned i = 0; i < W; ++i) w[i] = r[i];
    }
    if (count < (unsigned)N) {
#pragma unroll
        for (unsigned i = 0; i < W; ++i) {
            if constexpr (sizeof(T) == 2) w[i] = 2u * i + 1u < count ? w[i] : (2u * i < count ? w[i] & 0xffffu : 0u);
            else w[i] = i < count ? w[i] : 0u;
        }
    }
}

}  // namespace b200ccl::dev
