// The angle of a rotary pair, shared by rotary.hip and quantize.hip.
#pragma once

#include "dsa_common.h"

namespace dsa {
namespace rotary_core {

// cos and sin of position * frequency, times magnitude. The product and its
// reduction to a fraction of a turn are in 64 bits (in 32, the angle of position
// 163,839 would be off by 2^-7). What the fraction, within half a turn, loses in
// rounding to 32 bits, up to 2^-25 turns, is made up for to first order: it is more
// than what cos and sin themselves are off by.
__device__ __forceinline__ float2 turn(int64_t position, float frequency, float magnitude) {
  constexpr double kInverseTurn = 0.15915494309189533577;  // 1 / (2 pi)
  constexpr float kHalfTurn = 3.14159265358979323846f;
  const double turns = (double)position * (double)frequency * kInverseTurn;
  const double half_turns = 2.0 * (turns - __builtin_rint(turns));
  const float high = (float)half_turns;
  const float rest = kHalfTurn * (float)(half_turns - (double)high);
  float s, c;
  sincospif(high, &s, &c);
  return make_float2(__builtin_fmaf(-s, rest, c) * magnitude, __builtin_fmaf(c, rest, s) * magnitude);
}

// float32 -> bf16 bits, to nearest even (v_cvt_pk_bf16_f32; a NaN stays one).
__device__ __forceinline__ uint32_t to_bf16(float v) { return __builtin_bit_cast(uint16_t, (__bf16)v); }

// The position of a token: int32 or int64.
__device__ __forceinline__ int64_t position_at(const void* positions, int wide, int64_t token) {
  return wide ? static_cast<const int64_t*>(positions)[token] : static_cast<const int32_t*>(positions)[token];
}

}  // namespace rotary_core
}  // namespace dsa
