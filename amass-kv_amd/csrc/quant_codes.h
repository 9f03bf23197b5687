// Codes of the 8-bit cache (int8, e4m3) as 16-bit numbers, both exact: an int8 has at most 7
// significant bits and an e4m3 4, with exponents that fp16 and bf16 hold.
#pragma once

#include "../../include/amass_quant.h"
#include "common.h"

namespace amass {

typedef _Float16 half2_t __attribute__((ext_vector_type(2)));

// Four codes of a word, two 16-bit numbers a word.
//   e4m3        one conversion for two
//   int8, bf16  a conversion to fp32 for each (the byte is picked within it), whose upper half is
//               the bf16; 1.5 instructions a code
//   int8, fp16  1024 + u of the offset code u = code + 128 is a byte beside 0x64; less 1152: 1.25
template <int DT, int CT>
__device__ __forceinline__ void widen4(uint32_t x, uint32_t& lo, uint32_t& hi) {
    if constexpr (CT == AMASS_E4M3 && DT == AMASS_BF16) {
        lo = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(x, 1.f, false));
        hi = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(x, 1.f, true));
    } else if constexpr (CT == AMASS_E4M3) {
        lo = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(x, 1.f, false));
        hi = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(x, 1.f, true));
    } else if constexpr (DT == AMASS_BF16) {
        const auto f = [x](int n) { return __float_as_uint((float)(int8_t)(x >> (8 * n))); };
        lo = perm(f(1), f(0), 0x07060302u);
        hi = perm(f(3), f(2), 0x07060302u);
    } else {
        const uint32_t u = x ^ 0x80808080u;
        const half2_t back = {(_Float16)1152.f, (_Float16)1152.f};
        lo = __builtin_bit_cast(uint32_t, __builtin_bit_cast(half2_t, perm(0x64646464u, u, 0x04010400u)) - back);
        hi = __builtin_bit_cast(uint32_t, __builtin_bit_cast(half2_t, perm(0x64646464u, u, 0x04030402u)) - back);
    }
}

// code N of a word as fp32
template <int CT, int N>
__device__ __forceinline__ float code_f32(uint32_t x) {
    if constexpr (CT == AMASS_INT8) return (float)(int8_t)(x >> (8 * N));
    else return __builtin_amdgcn_cvt_f32_fp8(x, N);
}
template <int CT>
__device__ __forceinline__ float4 codes_f32(uint32_t x) {
    return make_float4(code_f32<CT, 0>(x), code_f32<CT, 1>(x), code_f32<CT, 2>(x), code_f32<CT, 3>(x));
}

// bit 7 of every byte that is an e4m3 NaN
__device__ __forceinline__ uint32_t nan_codes(uint32_t x) {
    return ((x & 0x7F7F7F7Fu) + 0x01010101u) & 0x80808080u;
}

template <int CT>
constexpr float MOST_CODE = CT == AMASS_INT8 ? 127.f : 448.f;

// Four quotients as codes, half to even, at most the largest (a NaN does not stay one).  int8: 1.5 2^23 + y has the
// whole number in its low byte.
template <int CT>
__device__ __forceinline__ uint32_t to_codes(float y0, float y1, float y2, float y3) {
    const auto cap = [](float y) { return fminf(fmaxf(y, -MOST_CODE<CT>), MOST_CODE<CT>); };
    if constexpr (CT == AMASS_INT8) {
        const auto byte = [&](float y) { return __float_as_uint(cap(y) + 12582912.f); };
        return perm(perm(byte(y3), byte(y2), 0x00000400u), perm(byte(y1), byte(y0), 0x00000400u), 0x05040100u);
    } else {
        const int lo = __builtin_amdgcn_cvt_pk_fp8_f32(cap(y0), cap(y1), 0, false);
        return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(cap(y2), cap(y3), lo, true);
    }
}

// least scale of a code type; the largest keeps code * scale finite
constexpr float LEAST_SCALE = 0x1p-64f;
template <int CT>
constexpr float MOST_SCALE = CT == AMASS_INT8 ? 0x1p121f : 0x1p119f;

// the scale that numbers of at most m take (m finite, m >= 0)
template <int CT>
__device__ __forceinline__ float step_of(float m) {
    float s;
    if constexpr (CT == AMASS_INT8) {
        s = __uint_as_float((__float_as_uint(m / 127.f) + 0xFFFFu) & 0xFFFF0000u);
    } else {
        const uint32_t u = __float_as_uint(m);                     // 448 = 1.75 2^8
        const int e = (int)(u >> 23) - 127 - 8 + ((u & 0x7FFFFFu) > 0x600000u ? 1 : 0);
        s = __uint_as_float((uint32_t)(max(e, -64) + 127) << 23);
    }
    return fminf(fmaxf(s, LEAST_SCALE), MOST_SCALE<CT>);
}

// x / s rounded to fp32, inv = 1 / s: the product is off by an ulp at most, its residual exact
__device__ __forceinline__ float quotient(float x, float s, float inv) {
    const float y = x * inv;
    return __builtin_fmaf(__builtin_fmaf(-y, s, x), inv, y);
}

// Four codes of scale `old` as those of scale s, inv = 1 / s.  An e4m3 NaN stays the code that it is: a cache that
// was quantised elsewhere may hold some, and rows that see one are NaN.
template <int CT>
__device__ __forceinline__ uint32_t round_again(uint32_t z, float old, float s, float inv) {
    const float4 f = codes_f32<CT>(z);
    const uint32_t c = to_codes<CT>(quotient(f.x * old, s, inv), quotient(f.y * old, s, inv),
                                    quotient(f.z * old, s, inv), quotient(f.w * old, s, inv));
    if constexpr (CT == AMASS_INT8) return c;
    const uint32_t nan = (nan_codes(z) >> 7) * 0xFFu;
    return (c & ~nan) | (z & nan);
}

}  // namespace amass
