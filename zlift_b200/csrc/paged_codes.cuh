// paged_codes.cuh -- 8-bit cache codes as 16-bit matrix operands, exactly.
#pragma once
#include "paged.h"

namespace zl {

// widen(u, lo, hi): the four codes in u as two pairs of 16-bit values (codes 0
// and 1 in lo, 2 and 3 in hi)
template <int ELEM, int CT>
struct Code {};                          // a 16-bit cache: nothing to widen

// int8 -> fp16: 0x6400 | (c + 128) is 1024 + 128 + c
template <>
struct Code<kF16, kI8> {
    static __device__ __forceinline__ void widen(uint32_t u, uint32_t& lo, uint32_t& hi) {
        const uint32_t x = u ^ 0x80808080u;
        const uint32_t k = 0x64806480u;              // 1152
        uint32_t a = __byte_perm(x, 0x64646464u, 0x4140), b = __byte_perm(x, 0x64646464u, 0x4342);
        const __half2 kh = *reinterpret_cast<const __half2*>(&k);
        const __half2 ah = __hsub2(*reinterpret_cast<__half2*>(&a), kh);
        const __half2 bh = __hsub2(*reinterpret_cast<__half2*>(&b), kh);
        lo = *reinterpret_cast<const uint32_t*>(&ah);
        hi = *reinterpret_cast<const uint32_t*>(&bh);
    }
};

// int8 -> bf16, whose 8 significant bits hold no offset of 128 beside 8 bits:
// with c = low7 - 128 * sign, (128 + low7) - (128 or 256, by the sign) = c
template <>
struct Code<kBF16, kI8> {
    static __device__ __forceinline__ uint32_t half(uint32_t y) {   // bytes c, 0x43, c, 0x43
        uint32_t a = y & 0xff7fff7fu, b = y & 0xff80ff80u;
        const __nv_bfloat162 r = __hsub2(*reinterpret_cast<__nv_bfloat162*>(&a),
                                         *reinterpret_cast<__nv_bfloat162*>(&b));
        return *reinterpret_cast<const uint32_t*>(&r);
    }
    static __device__ __forceinline__ void widen(uint32_t u, uint32_t& lo, uint32_t& hi) {
        lo = half(__byte_perm(u, 0x43434343u, 0x4140));
        hi = half(__byte_perm(u, 0x43434343u, 0x4342));
    }
};

// e4m3 -> fp16 by the hardware's conversion of two codes (exact; two
// instructions a word, where taking the halves apart in C++ cost more: drafted
// tokens 86 against 80 us)
template <>
struct Code<kF16, kE4M3> {
    static __device__ __forceinline__ void widen(uint32_t u, uint32_t& lo, uint32_t& hi) {
        asm("{\n\t.reg .b16 a, b;\n\tmov.b32 {a, b}, %2;\n\t"
            "cvt.rn.f16x2.e4m3x2 %0, a;\n\tcvt.rn.f16x2.e4m3x2 %1, b;\n\t}"
            : "=r"(lo), "=r"(hi) : "r"(u));
    }
};

// e4m3 -> bf16: sign, 4 exponent and 3 mantissa bits moved into place, which
// is 2^-120 of the code's value (the exponent biases differ by 120; subnormal
// codes become bf16 subnormals), brought back by an exact product
template <>
struct Code<kBF16, kE4M3> {
    static __device__ __forceinline__ uint32_t half(uint32_t p) {
        uint32_t x = (p & 0x80008000u) | ((p >> 4) & 0x07f007f0u);
        const uint32_t k = 0x7b807b80u;              // 2^120
        const __nv_bfloat162 r = __hmul2(*reinterpret_cast<__nv_bfloat162*>(&x),
                                         *reinterpret_cast<const __nv_bfloat162*>(&k));
        return *reinterpret_cast<const uint32_t*>(&r);
    }
    static __device__ __forceinline__ void widen(uint32_t u, uint32_t& lo, uint32_t& hi) {
        lo = half(__byte_perm(u, 0u, 0x1404));
        hi = half(__byte_perm(u, 0u, 0x3424));
    }
};

// fp16 weights carry their keys' V scales and a power of two `pow`, by which
// pow * (largest scale so far) stays in [256, 1024]: a weight of 2^kLazy8 (the
// most that a lazy maximum allows) does not overflow, and small scales keep
// their bits as far down as fp16 goes.
//
// A lazy maximum of 6 with [128, 512] took 587 us where this takes 594 (4 x 2048
// over 4096 tokens, int8), but sent rows whose weight sits on one token with a V
// 1000 times below the largest to be computed again (29 ms in place of 0.6).
constexpr float kLazy8 = 5.f;

// Takes the largest scale of the next keys; returns the factor by which the O
// summed so far has to be multiplied.  (Within 2^-90 and 2^90 the sums of 2^31
// weights stay in fp32's range.)
__device__ __forceinline__ float v_power(float big, float& most, float& pow) {
    if (!(big > most)) return 1.f;
    most = big;
    const float x = big * pow;
    if (x >= 256.f && x <= 1024.f) return 1.f;
    const int e = min(max(135 - (int)(__float_as_uint(big) >> 23), -90), 90);
    const float next = __uint_as_float((uint32_t)(127 + e) << 23);
    const float fix = next / pow;
    pow = next;
    return fix;
}

// log2 of a power of two
__device__ __forceinline__ float exponent_of(float pow) {
    return (float)((int)(__float_as_uint(pow) >> 23) - 127);
}

// A scale as a key for a maximum (`other` 0) or a minimum (all ones) over the
// keys that count: those with a scale of zero, none or a NaN do not, nor do
// infinities (which end in a NaN by themselves).
__device__ __forceinline__ uint32_t scale_key(float s, uint32_t other) {
    const uint32_t k = __float_as_uint(s) & 0x7fffffffu;
    return k - 1u < 0x7f7fffffu ? k : other;
}

// `pow` is one number for all keys of a tile, hidden ones and ones without
// weight among them, and a scale far below the largest leaves its weight
// among fp16's subnormals.  Where s * pow >= 1 for every scale, no weight
// loses more than an fp16 weight without a scale would.  Otherwise (`wide`) a row
// is looked at by its result: each of the n weights is off by 2^-25 at most
// beside its rounding, so O by n * 2^-25 * (largest code), and a row whose
// largest |O| (with pow in it) is not well above that is computed again
// (paged_finish.cuh) in fp32.
__device__ __forceinline__ bool wide_scales(uint32_t least, float most, float pow) {
    return __uint_as_float(least) * pow < 1.f || most * pow > 1024.f;
}
// what the largest |O| must reach: the loss is then below what rounding it to
// the output's type may cost
template <int ELEM, int CT>
__device__ __forceinline__ float trusted_from(int keys, float most, float pow) {
    constexpr float per_key = (CT == kI8 ? 128.f : 448.f) * 0x1p-25f * (ELEM == kBF16 ? 0x1p8f : 0x1p11f);
    return most * pow > 1024.f ? INFINITY : keys * per_key;
}

}  // namespace zl
