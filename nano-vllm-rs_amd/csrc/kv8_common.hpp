// kv8_common.hpp -- the number formats of the 8-bit KV cache (device side).
//
// A cached value is code * scale, with one scale per (block, kv head), K and V apart:
//   scale = 2^e, the smallest with max|x| <= top * 2^e   (0 for a block of zeros; e >= -126)
//   int8: top = 127, code an integer        E4M3 (OCP): top = 448, code one of its numbers
// Why a power of two and not max|x| / top, which would use the range to its end: x / scale, code *
// scale and the step from an old scale to a larger one are then exact, so (1) the only rounding of a
// value is the one to its code and a write has one right answer whatever order the work is done in,
// (2) a block that is filled token by token and whose scale grows on the way is off by less than one
// step of its final scale (1/2 + 1/4 + ... of it), where a free scale adds half a step at each growth,
// (3) E4M3 loses nothing in a growth but what leaves its smallest binade, and (4) codes times scale
// are exact in bf16 (from its smallest number on).  It costs int8 up to one bit, half a bit on average; E4M3 nothing.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

#include "nvllm_kernels.hpp"

namespace nvllm {
namespace kernels {
namespace kv8 {

typedef __attribute__((ext_vector_type(2))) unsigned u32x2;
typedef __attribute__((ext_vector_type(4))) unsigned u32x4;
typedef __attribute__((ext_vector_type(4))) float f32x4;
typedef __attribute__((ext_vector_type(2))) __bf16 bf16x2;

// Values past this are infinite to the cache: they take no part in a scale and saturate.  (One
// binade under the f32 limit, so that no code * scale overflows.)
constexpr float kHuge = 0x1p127f;

__device__ __forceinline__ float bf16_lo(unsigned w) { return __builtin_bit_cast(float, w << 16); }
__device__ __forceinline__ float bf16_hi(unsigned w) { return __builtin_bit_cast(float, w & 0xffff0000u); }
__device__ __forceinline__ unsigned pack_bf16x2(float lo, float hi) {
    bf16x2 r;
    r[0] = static_cast<__bf16>(lo);
    r[1] = static_cast<__bf16>(hi);
    return __builtin_bit_cast(unsigned, r);
}

// |x| where x counts towards a scale, 0 where it does not (infinite, NaN)
__device__ __forceinline__ float finite_abs(float x) {
    const float a = fabsf(x);
    return a <= kHuge ? a : 0.0f;
}

// scale of a block whose largest finite |x| is amax.  In the bits: the exponent of amax, plus one if
// its fraction exceeds that of top (127 = 1.984375 * 2^6, 448 = 1.75 * 2^8), minus top's exponent.
template <Kv8Format F> __device__ __forceinline__ float scale_of(float amax) {
    constexpr unsigned frac = F == Kv8Format::Int8 ? 0x7e0000u : 0x600000u;
    constexpr int top_exp = F == Kv8Format::Int8 ? 6 : 8;
    if (!(amax > 0.0f)) return 0.0f;
    int e = (int)((__builtin_bit_cast(unsigned, amax) + (0x7fffffu - frac)) >> 23) - top_exp;
    e = e < 1 ? 1 : e;  // no scale below 2^-126 (amax itself may be subnormal)
    return __builtin_bit_cast(float, (unsigned)e << 23);
}

// 1 / scale, exact (the exponent field e becomes 254 - e; e = 1 .. 249); 1 for the scale 0, whose
// block holds nothing but zeros, infinities and NaN
__device__ __forceinline__ float inverse_scale(float s) {
    return s > 0.0f ? __builtin_bit_cast(float, (254u << 23) - __builtin_bit_cast(unsigned, s)) : 1.0f;
}

// y = x / scale of four values -> four codes (byte i = code of y[i]), to nearest, ties to even.
// Infinities saturate; a NaN becomes E4M3's NaN, and 0 in int8, which has none.
template <Kv8Format F> __device__ __forceinline__ unsigned encode4(float y0, float y1, float y2, float y3) {
    constexpr float top = F == Kv8Format::Int8 ? 127.0f : 448.0f;
    if constexpr (F == Kv8Format::Int8) {
        // adding 1.5 * 2^23 rounds to an integer and leaves it, two's complement, in the low bits
        const auto enc = [&](float y) -> unsigned {
            y = y == y ? y : 0.0f;
            return __builtin_bit_cast(unsigned, fminf(fmaxf(y, -top), top) + 12582912.0f);
        };
        const unsigned a = __builtin_amdgcn_perm(enc(y1), enc(y0), 0x0c0c0400u);
        const unsigned b = __builtin_amdgcn_perm(enc(y3), enc(y2), 0x04000c0cu);
        return a | b;
    } else {
        const auto clip = [&](float y) -> float { return y == y ? fminf(fmaxf(y, -top), top) : y; };
        int w = __builtin_amdgcn_cvt_pk_fp8_f32(clip(y0), clip(y1), 0, false);
        return (unsigned)__builtin_amdgcn_cvt_pk_fp8_f32(clip(y2), clip(y3), w, true);
    }
}

// byte `i` of w as a number
template <Kv8Format F> __device__ __forceinline__ void decode4(unsigned w, float *x) {
    if constexpr (F == Kv8Format::Int8) {
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = (float)(signed char)(w >> (8 * i));
    } else {
        const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, false);
        const auto hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, true);
        x[0] = lo[0];
        x[1] = lo[1];
        x[2] = hi[0];
        x[3] = hi[1];
    }
}

template <Kv8Format F> __device__ __forceinline__ float decode1(unsigned char c) {
    float x[4];
    decode4<F>(c, x);
    return x[0];
}
template <Kv8Format F> __device__ __forceinline__ unsigned char encode1(float y) {
    return (unsigned char)encode4<F>(y, 0.0f, 0.0f, 0.0f);
}

// y to 24 bits, to odd: truncated, and the last bit set where that lost something.  A later rounding to a
// code then falls as if from y itself (rounding to nearest here would put 1 value in 2^17 on the wrong
// side of a code's border).
__device__ __forceinline__ float narrow_odd(double y) {
    const float f = (float)y;
    const double d = (double)f;
    unsigned u = __builtin_bit_cast(unsigned, f);
    if (d != y && y == y) {
        if (fabs(d) > fabs(y)) u -= 1;  // (an infinity, from a y past f32's range, becomes the largest number)
        u |= 1;
    }
    return __builtin_bit_cast(float, u);
}
__device__ __forceinline__ float narrow_odd(float y) { return y; }
template <Kv8Format F> __device__ __forceinline__ unsigned char encode1(double y) { return encode1<F>(narrow_odd(y)); }

// the codes of a kept row under a larger scale (ratio = old / new, a power of two <= 1/2).  A code
// that is no number of the format (int8's -128, which no write makes) is brought back into range.
template <Kv8Format F> __device__ __forceinline__ unsigned rescale4(unsigned w, float ratio) {
    float x[4];
    decode4<F>(w, x);
    return encode4<F>(x[0] * ratio, x[1] * ratio, x[2] * ratio, x[3] * ratio);
}

__device__ __forceinline__ float wave_max(float x) {
#pragma unroll
    for (int m = 32; m > 0; m >>= 1) x = fmaxf(x, __shfl_xor(x, m));
    return x;
}

template <typename ET> __device__ __forceinline__ float to_f32(ET x) { return static_cast<float>(x); }

}  // namespace kv8
}  // namespace kernels
}  // namespace nvllm
