// The 8-bit cache: codes, their powers of two, and where they lie in a block.
//
// A value x of a (16-token block, kv head) is held as a code c, x ~ c 2^e, with
// one exponent e for the block's keys and one for its values.  e is the least
// whole number (at least kQ8LeastExponent) with |x| <= kQ8Largest 2^e for every
// x of the block, and c is x 2^-e rounded to the nearest code, ties to
// even.  A power of two in place of amax / largest costs up to one bit of the
// integer codes (none of the floating ones), and buys exactness: dividing by it
// and multiplying with it round nothing, so a block whose exponent grows with an
// appended row is rounded again only where bits fall off, the attention applies
// it to the f32 scores and weights without an error, and every rounding decision
// is the same on any machine.  Infinite values are taken as fp16's largest, 65504
// (left out of the exponent, they would shrink to the size of what is around
// them); NaN sets no exponent and becomes the e4m3 NaN, or 0 in int8, which has
// none.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

#include "pvlc_device.hpp"
#include "pvlc_internal.hpp"

namespace pvlc {

typedef uint32_t q8x4_t __attribute__((ext_vector_type(4)));  // 16 codes
typedef _Float16 half2_t __attribute__((ext_vector_type(2)));
typedef float float2_t __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2_t __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));

// 2^e, -126 <= e <= 127.
__device__ inline float exp2_whole(int e) { return __uint_as_float(static_cast<uint32_t>(e + 127) << 23); }

// An fp16 value as it is held: infinities are 65504.
__device__ inline float q8_value(float x) { return x != x ? x : __builtin_amdgcn_fmed3f(x, -65504.f, 65504.f); }
// The larger of a size and that of such a value (a NaN changes nothing).
__device__ inline float q8_size(float size, float x) { return fmaxf(size, __builtin_fabsf(x)); }

// The exponent for sizes up to amax (0 or an fp16 value's size, so never a
// subnormal f32): with amax = 1.f 2^k, 448 is 1.75 2^8
// and 127 is 1.984375 2^6.
template <int CODE>
__device__ inline int q8_exponent(float amax) {
    const uint32_t bits = __float_as_uint(amax);
    const int k = static_cast<int>(bits >> 23) - 127;
    const uint32_t fraction = bits & 0x7FFFFFu;
    const int e = CODE == PVLC_HIP_KV_E4M3 ? k - 8 + (fraction > 0x600000u) : k - 6 + (fraction > 0x7E0000u);
    return max(e, kQ8LeastExponent);
}

// Four values, divided by the block's power (so at most the largest code in
// size, or NaN), to four codes.
template <int CODE>
__device__ inline uint32_t q8_encode(float a, float b, float c, float d) {
    if constexpr (CODE == PVLC_HIP_KV_E4M3) {
        const int r = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
        return static_cast<uint32_t>(__builtin_amdgcn_cvt_pk_fp8_f32(c, d, r, true));
    } else {
        auto code = [](float x) { return static_cast<uint32_t>(static_cast<int>(x != x ? 0.f : __builtin_rintf(x))) & 0xFFu; };
        return code(a) | code(b) << 8 | code(c) << 16 | code(d) << 24;
    }
}

// Four codes as f32.
template <int CODE>
__device__ inline float4_t q8_decode(uint32_t w) {
    if constexpr (CODE == PVLC_HIP_KV_E4M3) {
        const float2_t lo = __builtin_amdgcn_cvt_pk_f32_fp8(static_cast<int>(w), false);
        const float2_t hi = __builtin_amdgcn_cvt_pk_f32_fp8(static_cast<int>(w), true);
        return float4_t{lo[0], lo[1], hi[0], hi[1]};
    } else {
        return float4_t{static_cast<float>(static_cast<int8_t>(w)), static_cast<float>(static_cast<int8_t>(w >> 8)),
                        static_cast<float>(static_cast<int8_t>(w >> 16)), static_cast<float>(static_cast<int8_t>(w >> 24))};
    }
}

// Four codes of a block whose exponent grew by `grown` >= 0, rounded again.
template <int CODE>
__device__ inline uint32_t q8_requantise(uint32_t w, int grown) {
    // (a power below the least normal one only for codes that all round to 0)
    const float4_t v = q8_decode<CODE>(w) * exp2_whole(-min(grown, 126));
    return q8_encode<CODE>(v[0], v[1], v[2], v[3]);
}

// Eight codes as fp16, exactly: an MFMA operand.  e4m3 by the part's own
// conversion; int8 by way of 1024 + (c + 128), which fp16 holds exactly with
// the byte as its low bits, so a byte permutation builds two of them.
template <int CODE>
__device__ inline half8_t q8_half8(uint32_t lo, uint32_t hi) {
    half8_t r;
    if constexpr (CODE == PVLC_HIP_KV_E4M3) {
        const half2_t a = __builtin_bit_cast(half2_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, 1.f, false));
        const half2_t b = __builtin_bit_cast(half2_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, 1.f, true));
        const half2_t c = __builtin_bit_cast(half2_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, 1.f, false));
        const half2_t d = __builtin_bit_cast(half2_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, 1.f, true));
        r = half8_t{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
    } else {
        const half2_t zero = {static_cast<_Float16>(1152.f), static_cast<_Float16>(1152.f)};
        half2_t h[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t u = (i < 2 ? lo : hi) ^ 0x80808080u;
            // bytes {u[2j], 0x64, u[2j + 1], 0x64}: 4 selects the other operand's byte 0
            h[i] = __builtin_bit_cast(half2_t, __builtin_amdgcn_perm(0x64646464u, u, i & 1 ? 0x04030402u : 0x04010400u)) - zero;
        }
        r = half8_t{h[0][0], h[0][1], h[1][0], h[1][1], h[2][0], h[2][1], h[3][0], h[3][1]};
    }
    return r;
}

// Eight codes as bf16, exactly (at most 8 significant bits): an MFMA operand.  int8
// by way of f32, whose low half is 0 then.
template <int CODE>
__device__ inline bf16x8_t q8_bf16x8(uint32_t lo, uint32_t hi) {
    q8x4_t r;
    if constexpr (CODE == PVLC_HIP_KV_E4M3) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const uint32_t w = i ? hi : lo;
            r[i * 2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.f, false));
            r[i * 2 + 1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.f, true));
        }
    } else {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const float4_t x = q8_decode<CODE>(i ? hi : lo);
            // the high halves of two
            r[i * 2] = __builtin_amdgcn_perm(__float_as_uint(x[1]), __float_as_uint(x[0]), 0x07060302u);
            r[i * 2 + 1] = __builtin_amdgcn_perm(__float_as_uint(x[3]), __float_as_uint(x[2]), 0x07060302u);
        }
    }
    return __builtin_bit_cast(bf16x8_t, r);
}

// The largest of the 64 lanes, in every lane (see wave_sum).
__device__ inline float wave_max(float v) {
    v = fmaxf(v, dpp_f32<0xB1>(v));
    v = fmaxf(v, dpp_f32<0x4E>(v));
    v = fmaxf(v, dpp_f32<0x124>(v));
    v = fmaxf(v, dpp_f32<0x128>(v));
    float m = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), 0));
#pragma unroll
    for (int l = 16; l < 64; l += 16) m = fmaxf(m, __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), l)));
    return m;
}

}  // namespace pvlc
