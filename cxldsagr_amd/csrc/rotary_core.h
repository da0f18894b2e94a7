// The angle of a rotary pair, shared by rotary.hip and quantize.hip.
#pragma once

#include "dsa_common.h"

namespace dsa {
namespace rotary_core {

// cos and sin of position * frequency, times magnitude. The product and its
// reduction to a fraction of a turn are in 64 bits (in 32, the angle of position
// 163,839 would be off by 2^-7); the fraction, within half a turn, is rounded to
// 32 bits, which moves the angle by at most 2^-25 turns.
__device__ __forceinline__ float2 turn(int64_t position, float frequency, float magnitude) {
  constexpr double kInverseTurn = 0.15915494309189533577;  // 1 / (2 pi)
  const double turns = (double)position * (double)frequency * kInverseTurn;
  const float half_turns = 2.0f * (float)(turns - __builtin_rint(turns));
  float s, c;
  sincospif(half_turns, &s, &c);
  return make_float2(c * magnitude, s * magnitude);
}

// float32 -> bf16 bits, to nearest even (v_cvt_pk_bf16_f32; a NaN stays one).
__device__ __forceinline__ uint32_t to_bf16(float v) { return __builtin_bit_cast(uint16_t, (__bf16)v); }

// The position of a token: int32 or int64.
__device__ __forceinline__ int64_t position_at(const void* positions, int wide, int64_t token) {
  return wide ? static_cast<const int64_t*>(positions)[token] : static_cast<const int32_t*>(positions)[token];
}

}  // namespace rotary_core
}  // namespace dsa
