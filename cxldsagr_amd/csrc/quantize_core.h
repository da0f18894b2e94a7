// The quantisation rule of e4m3 rows, shared by every kernel that writes them:
// scale = amax * fl32(1/448), as a power of two where ue8m0, codes of the clamped
// quotients rounded to nearest even.
#pragma once

#include "dsa_common.h"

namespace dsa {
namespace {

template <int kWidth>
__device__ __forceinline__ uint32_t max_abs_bits_reduce(uint32_t v) {
  // |x| as fp32 bits orders like the magnitude; any NaN (bits > 0x7F800000)
  // wins, which is the NaN-propagating max the reference uses.
#pragma unroll
  for (int offset = kWidth / 2; offset > 0; offset >>= 1) {
    uint32_t o = __shfl_xor(v, offset, kWidth);
    v = v > o ? v : o;
  }
  return v;
}

__device__ __forceinline__ float scale_from_amax_bits(uint32_t amax_bits, bool ue8m0) {
  uint32_t bits;
  if (amax_bits > 0x7F800000u) {
    bits = kCanonicalNan;
  } else {
    float amax = fmaxf(__uint_as_float(amax_bits), 1e-4f);
    bits = __float_as_uint(amax * kReciprocal448);
    if (ue8m0) bits = (bits + 0x7FFFFFu) & 0x7F800000u;
  }
  return __uint_as_float(bits);
}

__device__ __forceinline__ uint32_t quantize_one(float v, float scale, float inverse, bool ue8m0) {
  float y = ue8m0 ? v * inverse : __fdiv_rn(v, scale);
  if (y != y) return 0x7Fu;
  y = fminf(fmaxf(y, -448.0f), 448.0f);
  return f32_to_e4m3fn(y);
}

// Codes of v[0 .. 7] of a row with the given scale, in two words. With a finite
// scale every value is finite and the hardware conversion of the clamped
// quotients gives f32_to_e4m3fn's codes (equal on every fp32 value of
// magnitude up to 448); the software encoding (~20 instructions a value, what
// bound the bulk packs) is left with rows that hold an infinity or a NaN.
// 65536 history rows (index K and KV, 144 MB moved, 27.5 us at the rate of a
// large copy): 43.0 -> 33.9 us together with the one launch for both.
__device__ __forceinline__ void quantize_eight(const float (&v)[8], float scale, bool ue8m0,
                                               uint32_t& lo, uint32_t& hi) {
  const uint32_t bits = __float_as_uint(scale);
  if ((bits & 0x7F800000u) == 0x7F800000u) {
    const float inverse = 1.0f / scale;
    lo = hi = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      lo |= quantize_one(v[i], scale, inverse, ue8m0) << (8 * i);
      hi |= quantize_one(v[4 + i], scale, inverse, ue8m0) << (8 * i);
    }
    return;
  }
  // A UE8M0 scale is a power of two (2^-22 .. 2^120): its exact reciprocal.
  const float inverse = __uint_as_float(0x7F000000u - bits);
  float y[8];
#pragma unroll
  for (int i = 0; i < 8; ++i)
    y[i] = __builtin_amdgcn_fmed3f(ue8m0 ? v[i] * inverse : __fdiv_rn(v[i], scale), -448.0f, 448.0f);
  lo = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(y[0], y[1], 0, false);
  lo = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(y[2], y[3], (int)lo, true);
  hi = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(y[4], y[5], 0, false);
  hi = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(y[6], y[7], (int)hi, true);
}

}  // namespace
}  // namespace dsa
