// What the kernels of the 8-bit cache share: the two code types, their conversion to half precision, and the scale of a block.
//
// A block is one page of one key/value head (keys and values apart).  It holds codes c and one float32 scale s; the cached
// number is c * s.  s is the smallest power of two with max|x| <= largest code * s, for two reasons.  A block that grows while
// a request decodes is brought to its new scale by c * (s / s'), a power of two: for e4m3 that is exact as long as the code
// stays a normal number, and for int8 the errors of all such steps together stay below one step of the new scale (1/2 + 1/4 +
// ...), where scales in small steps would add half a step each time.  And c * s is a bfloat16 number without rounding (at most
// seven significant bits).  It costs e4m3 nothing (its steps are relative); int8 loses up to one bit of its seven.
// What is not finite has no code: a block that is given such a value gets a scale of NaN, and reads as NaN as a whole.
#pragma once

#include <cuda_fp16.h>

#include "common.cuh"

enum SandyCode : int { SANDY_E4M3 = 0, SANDY_INT8 = 1 };

namespace {

constexpr int SMALLEST_SCALE_EXPONENT = -100;             // what a block of zeros has
constexpr unsigned LARGEST_KEPT_BITS = 0x7f700000u;       // 1.875 * 2^127: above it a rounded code times its scale is infinite

// Bits of the scale for a block whose largest |x| has the bits `amax` (finite, at most LARGEST_KEPT_BITS).
template <int CODE>
__device__ __forceinline__ float scale_for(unsigned amax) {
    // the largest code is 1.75 * 2^8 (e4m3) or 1.984375 * 2^6 (int8)
    constexpr int TOP = CODE == SANDY_E4M3 ? 8 : 6;
    constexpr unsigned MANTISSA = CODE == SANDY_E4M3 ? 0x600000u : 0x7e0000u;
    const int e = (int)(amax >> 23) - 127 - TOP + ((amax & 0x7fffffu) > MANTISSA ? 1 : 0);
    return __uint_as_float((unsigned)(max(e, SMALLEST_SCALE_EXPONENT) + 127) << 23);
}

// Four numbers, times inv, as four codes (the first in the low byte).  Round to nearest, ties to even; |x * inv| at most the largest code.
template <int CODE>
__device__ __forceinline__ unsigned encode4(float a, float b, float c, float d, float inv) {
    if (CODE == SANDY_E4M3) {
        unsigned r;
        asm("{\n\t.reg .b16 l, h;\n\tcvt.rn.satfinite.e4m3x2.f32 l, %2, %1;\n\tcvt.rn.satfinite.e4m3x2.f32 h, %4, %3;\n\tmov.b32 %0, {l, h};\n\t}"
            : "=r"(r)
            : "f"(a * inv), "f"(b * inv), "f"(c * inv), "f"(d * inv));
        return r;
    }
    // 1.5 * 2^23 added: the last place is 1, so the sum is rounded to a whole number, which is its low byte
    const unsigned p = __float_as_uint(fmaf(a, inv, 12582912.0f)), q = __float_as_uint(fmaf(b, inv, 12582912.0f));
    const unsigned r = __float_as_uint(fmaf(c, inv, 12582912.0f)), s = __float_as_uint(fmaf(d, inv, 12582912.0f));
    return __byte_perm(__byte_perm(p, q, 0x0040), __byte_perm(r, s, 0x0040), 0x5410);
}

// Four codes as two pairs of half-precision numbers: bytes 0, 1 and bytes 2, 3.  Exact for every code.
template <int CODE>
__device__ __forceinline__ void decode4(unsigned w, unsigned& lo, unsigned& hi) {
    if (CODE == SANDY_E4M3) {
        asm("{\n\t.reg .b16 a, b;\n\tmov.b32 {a, b}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, a;\n\tcvt.rn.f16x2.e4m3x2 %1, b;\n\t}"
            : "=r"(lo), "=r"(hi)
            : "r"(w));
    } else {
        // c + 128 as the low byte of the half 1024 + (c + 128), then 1152 off
        const unsigned u = w ^ 0x80808080u;
        const unsigned a = __byte_perm(u, 0x64646464u, 0x4140), b = __byte_perm(u, 0x64646464u, 0x4342);
        const __half2 off = __floats2half2_rn(1152.0f, 1152.0f);
        const __half2 x = __hsub2(*reinterpret_cast<const __half2*>(&a), off), y = __hsub2(*reinterpret_cast<const __half2*>(&b), off);
        lo = *reinterpret_cast<const unsigned*>(&x);
        hi = *reinterpret_cast<const unsigned*>(&y);
    }
}

// tanh for scores under a cap.  Near 0 1 - 2 / (1 + e^2x) keeps an error of 2^-22, which a large cap multiplies: at 10^6, a quarter of a nat.
// There the series, off by 62/2835 x^8 of the result (2^-29 at an eighth).
__device__ __forceinline__ float tanh_capped(float x) {
    const float y = x * x;
    const float near = x * fmaf(y, fmaf(y, fmaf(y, -17.0f / 315.0f, 2.0f / 15.0f), -1.0f / 3.0f), 1.0f);
    return y < 1.0f / 64.0f ? near : tanh_fast(x);
}

__device__ __forceinline__ float2 half2_floats(unsigned h) { return __half22float2(*reinterpret_cast<const __half2*>(&h)); }

}  // namespace
