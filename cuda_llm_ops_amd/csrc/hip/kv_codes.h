// 8-bit cache codes on the device: widening to the MFMA types, scaling and
// rounding (gfx950).
#pragma once

#include "fgqa_device.h"

namespace fgqa {

typedef _Float16 f16x8_t __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2_t __attribute__((ext_vector_type(2)));

enum KvCode { kCodeBf16 = 0, kCodeFp8 = 1, kCodeInt8 = 2 };

constexpr float kFp8Max = 448.f;
constexpr float kInt8Max = 127.f;
constexpr float kLargest = 3.40282347e38f;   // of fp32

// Byte i of w as a signed number.
template <int i>
__device__ __forceinline__ float int8_of(uint32_t w) {
    return (float)(int)(int8_t)(w >> (8 * i));
}

// 8 codes -> 8 bf16, exactly: e4m3 values have 4 significant bits and int8 ones
// up to 8, as bf16 has, so the int8 numbers' upper halves as floats are theirs.
template <int kCode>
__device__ __forceinline__ bf16x8_t codes_to_bf16(uint32_t w0, uint32_t w1) {
    u32x4_t r;
    if constexpr (kCode == kCodeFp8) {
        r[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w0, 1.0f, false));
        r[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w0, 1.0f, true));
        r[2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w1, 1.0f, false));
        r[3] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w1, 1.0f, true));
    } else {
        auto pair = [](float lo, float hi) {
            return __builtin_amdgcn_perm(__float_as_uint(hi), __float_as_uint(lo), 0x07060302u);
        };
        r[0] = pair(int8_of<0>(w0), int8_of<1>(w0));
        r[1] = pair(int8_of<2>(w0), int8_of<3>(w0));
        r[2] = pair(int8_of<0>(w1), int8_of<1>(w1));
        r[3] = pair(int8_of<2>(w1), int8_of<3>(w1));
    }
    return as_bf16x8(r);
}

// 8 codes -> 8 fp16, exactly.  int8: a byte u = code + 128 under 0x64 is the
// fp16 number 1024 + u, and 1024 + u - 1152 = code has no rounding.
template <int kCode>
__device__ __forceinline__ f16x8_t codes_to_f16(uint32_t w0, uint32_t w1) {
    u32x4_t r;
    if constexpr (kCode == kCodeFp8) {
        r[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w0, 1.0f, false));
        r[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w0, 1.0f, true));
        r[2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w1, 1.0f, false));
        r[3] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w1, 1.0f, true));
    } else {
        const f16x2_t off = {(_Float16)1152.f, (_Float16)1152.f};
        auto pair = [&](uint32_t u, uint32_t sel) {
            const uint32_t biased = __builtin_amdgcn_perm(0x64646464u, u, sel);
            return __builtin_bit_cast(uint32_t, __builtin_bit_cast(f16x2_t, biased) - off);
        };
        const uint32_t u0 = w0 ^ 0x80808080u, u1 = w1 ^ 0x80808080u;
        r[0] = pair(u0, 0x04010400u);
        r[1] = pair(u0, 0x04030402u);
        r[2] = pair(u1, 0x04010400u);
        r[3] = pair(u1, 0x04030402u);
    }
    return __builtin_bit_cast(f16x8_t, r);
}

// 4 codes of w -> their values before scaling.
template <int kCode>
__device__ __forceinline__ f32x4_t codes_to_f32(uint32_t w) {
    if constexpr (kCode == kCodeFp8) {
        const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8(w, false);
        const auto hi = __builtin_amdgcn_cvt_pk_f32_fp8(w, true);
        return f32x4_t{lo[0], lo[1], hi[0], hi[1]};
    } else {
        return f32x4_t{int8_of<0>(w), int8_of<1>(w), int8_of<2>(w), int8_of<3>(w)};
    }
}

// The smallest power of two s >= 2^-126 with amax <= s * (the codes' largest):
// 448 = 1.75 * 2^8, 127 = 1.984375 * 2^6, so one comparison of amax's
// significand decides the exponent.
template <int kCode>
__device__ __forceinline__ float block_scale(float amax) {
    constexpr uint32_t kTop = kCode == kCodeFp8 ? 0x600000u : 0x7e0000u;
    constexpr int kExp = kCode == kCodeFp8 ? 8 : 6;
    const uint32_t bits = __float_as_uint(amax);
    const int e = (int)(bits >> 23) - kExp + ((bits & 0x7fffffu) > kTop ? 1 : 0);   // biased by 127
    return __uint_as_float((uint32_t)max(e, 1) << 23);
}

// 4 scaled values -> 4 codes, to nearest even, saturated; NaN: e4m3's NaN, int8 0.
template <int kCode>
__device__ __forceinline__ uint32_t to_codes(f32x4_t y) {
    if constexpr (kCode == kCodeFp8) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float c = fminf(fmaxf(y[i], -kFp8Max), kFp8Max);
            y[i] = y[i] == y[i] ? c : y[i];
        }
        const int lo = __builtin_amdgcn_cvt_pk_fp8_f32(y[0], y[1], 0, false);
        return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(y[2], y[3], lo, true);
    } else {
        uint32_t w = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float c = fminf(fmaxf(__builtin_rintf(y[i]), -kInt8Max), kInt8Max);
            const int n = y[i] == y[i] ? (int)c : 0;
            w |= ((uint32_t)n & 0xffu) << (8 * i);
        }
        return w;
    }
}

// 16 finite bf16 values (two 16-byte pieces) / s -> 16 codes, for a power of two s
// that brings them inside the codes' range, so nothing saturates: x / s is exact
// and rounds once.  e4m3: the conversion divides by the power of two itself.
// int8: 1.5 * 2^23 + x / s rounds to a whole number whose low byte is the code.
template <int kCode>
__device__ __forceinline__ u32x4_t finite_to_codes(const u32x4_t (&x)[2], float s, float inv) {
    u32x4_t r;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t w0 = x[i / 2][2 * (i % 2)], w1 = x[i / 2][2 * (i % 2) + 1];
        if constexpr (kCode == kCodeFp8) {
            typedef short s16x2_t __attribute__((ext_vector_type(2)));
            s16x2_t c = {0, 0};
            c = __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(c, __builtin_bit_cast(bf16x2_t, w0), s, false);
            c = __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(c, __builtin_bit_cast(bf16x2_t, w1), s, true);
            r[i] = __builtin_bit_cast(uint32_t, c);
        } else {
            const float magic = 12582912.f;
            const uint32_t a = __float_as_uint(fmaf(__uint_as_float(w0 << 16), inv, magic));
            const uint32_t b = __float_as_uint(fmaf(__uint_as_float(w0 & 0xffff0000u), inv, magic));
            const uint32_t c = __float_as_uint(fmaf(__uint_as_float(w1 << 16), inv, magic));
            const uint32_t d = __float_as_uint(fmaf(__uint_as_float(w1 & 0xffff0000u), inv, magic));
            r[i] = __builtin_amdgcn_perm(__builtin_amdgcn_perm(d, c, 0x0c0c0400u), __builtin_amdgcn_perm(b, a, 0x0c0c0400u),
                                         0x05040100u);
        }
    }
    return r;
}

// Over the wave's four groups of 16 lanes, in every lane: v_permlane16_swap and
// v_permlane32_swap, without the LDS round trips of a shuffle.
__device__ __forceinline__ float groups_max(float v) {
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return half_max(fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1])));
}
__device__ __forceinline__ float groups_sum(float v) {
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return half_sum(__uint_as_float(r[0]) + __uint_as_float(r[1]));
}

__device__ __forceinline__ float finite_abs(float x) {
    const float a = fabsf(x);
    return a < INFINITY ? a : 0.f;   // (false for NaN)
}

// |x| of a code times a scale, NaN as 0.  Codes are finite, so an infinite product is
// a number past fp32's largest: the largest bf16 number, 1.992 * 2^127, is held as
// 2^128.  It counts as the largest, whose scale is the same.
__device__ __forceinline__ float capped_abs(float x) {
    return x == x ? fminf(fabsf(x), kLargest) : 0.f;
}

}  // namespace fgqa
