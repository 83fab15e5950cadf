// Eight-bit floating point (e4m3: sign, four bits of exponent, three of mantissa, to 448, no infinities) with a
// binary32 scale for each block of 128 values.
//
// For a block with the largest magnitude t: s = max(t / 448, 2^-126), and a value x becomes the e4m3 nearest to
// x * (1 / s), ties to the even code, each of the two divisions and the product rounded to binary32 once.  The
// product is at most 448 (1 + 2^-22), which rounds to 448.  A block with an infinity or a NaN has s = NaN and
// NaN codes throughout, so that what is computed from it is NaN.
#pragma once
#include "lsk_common.h"

namespace lsk {

struct Fp8Scale {
  float s, inv;
};
LSK_DEV Fp8Scale fp8_scale(uint32_t top) {  // top: the bits of the largest magnitude, as an integer
  const float t = __uint_as_float(top);
  float s = f32_div(t, 448.0f);
  s = s < 0x1p-126f ? 0x1p-126f : s;
  if (top >= 0x7f800000u) s = __uint_as_float(0x7fc00000u);
  return {s, f32_div(1.0f, s)};
}

// The larger of the 16 lanes of a DPP row, in each of them.
LSK_DEV uint32_t row_max_u32(uint32_t v) {
  auto up = [&](uint32_t o) { v = v > o ? v : o; };
  up((uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0xb1, 0xf, 0xf, false));   // quad [1,0,3,2]
  up((uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x4e, 0xf, 0xf, false));   // quad [2,3,0,1]
  up((uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x141, 0xf, 0xf, false));  // half-row mirror
  up((uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x140, 0xf, 0xf, false));  // row mirror
  return v;
}

// (magnitudes compare like their bits; a NaN's are above infinity's)
LSK_DEV uint32_t top8(const float (&v)[8]) {
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const uint32_t u = __float_as_uint(v[i]) & 0x7fffffffu;
    top = top > u ? top : u;
  }
  return top;
}

// Eight values times inv as e4m3 bytes, the first lowest (v_cvt_pk_fp8_f32 rounds to nearest, ties to even,
// subnormals kept, a NaN to 0x7f: compared with the definition over every border of every code).
LSK_DEV uint2 quantize8_fp8(const float (&v)[8], float inv) {
  auto four = [&](int i) {
    int w = __builtin_amdgcn_cvt_pk_fp8_f32(f32_mul(v[i], inv), f32_mul(v[i + 1], inv), 0, false);
    return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(f32_mul(v[i + 2], inv), f32_mul(v[i + 3], inv), w, true);
  };
  return make_uint2(four(0), four(4));
}

// A block of 128 values held eight a lane by a DPP row of 16 lanes: its codes and scale.
LSK_DEV uint2 quantize_row_fp8(const float (&v)[8], float& scale) {
  const Fp8Scale s = fp8_scale(row_max_u32(top8(v)));
  scale = s.s;
  return quantize8_fp8(v, s.inv);
}

}  // namespace lsk
