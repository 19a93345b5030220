// hx_f8.hpp -- values in 8-bit floating point (e4m3: 4 exponent bits, 3 mantissa bits, largest value 448) with a scale for each
// block of 128.
//
//   a = max(largest |v| of the block, 2^-100)    scale = a / 448    code = e4m3(v * (448 / a)), rounded to nearest even
//
// 448 / a and the products are single fp32 operations, so |v * (448 / a)| is at most 448 (1 + 2^-23), which rounds to 448.  The
// floor keeps 448 / a finite; a block of zeros has codes 0.  A NaN or an infinity makes the scale NaN or infinite and with it every value
// that the block stands for NaN: codes are NaN, or 0 times an infinite scale.
#pragma once
#include "hx_f8_plan.hpp"
#include "hx_gemv.hpp"

namespace hx {

constexpr float F8_TOP = 448.0f, F8_TINY = 0x1p-100f;

// Largest of a u32 over each row of 16 lanes, in all of them.
HX_INLINE uint32_t f8_row_max(uint32_t v)
{
    v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x128, 0xf, 0xf, false));  // row_ror:8
    v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x124, 0xf, 0xf, false));
    v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x122, 0xf, 0xf, false));
    return max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x121, 0xf, 0xf, false));
}

// Bits of |v|: they compare as the values do, and a NaN's are above all others'.
HX_INLINE uint32_t f8_abs_bits(float v) { return __builtin_bit_cast(uint32_t, v) & 0x7fffffffu; }

// Factor and scale of a block whose largest |v| has these bits.
struct F8Scale {
    float factor, scale;
};
HX_INLINE F8Scale f8_scale(uint32_t bits)
{
    const float a = __builtin_bit_cast(float, max(bits, __builtin_bit_cast(uint32_t, F8_TINY)));
    return {F8_TOP / a, a / F8_TOP};
}

// Codes of four values, the first in the low byte.
HX_INLINE uint32_t f8_codes(float a, float b, float c, float d)
{
    const int lo = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
    return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, lo, true);
}

}  // namespace hx
