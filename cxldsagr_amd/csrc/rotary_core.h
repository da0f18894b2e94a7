// The angle of a rotary pair, shared by rotary.hip and quantize.hip.
#pragma once

#include "dsa_common.h"

namespace dsa {
namespace rotary_core {

// cos and sin of position * frequency, times magnitude, in 64 bits and rounded once to 32
// (in 32, the angle of position 163,839 would be off by 2^-7; a magnitude in 32 bits would
// add a rounding of its own). The angle in turns, less
// whole turns and quarters, leaves x within an eighth of a turn, where the power series
// of sin to x^11 and of cos to x^10 are off by less than 2^-32: fewer instructions than
// 32-bit functions of any angle take, whose results were off by up to 2^-23.
__device__ __forceinline__ float2 turn(int64_t position, float frequency, double magnitude) {
  constexpr double kInverseTurn = 0.15915494309189533577, kTurn = 6.28318530717958647693;  // 1 / (2 pi), 2 pi
  const double turns = (double)position * (double)frequency * kInverseTurn;
  const double part = turns - __builtin_rint(turns);
  const double quarters = __builtin_rint(4.0 * part);
  const double x = kTurn * __builtin_fma(-0.25, quarters, part), z = x * x;
  double s = -1.0 / 39916800;
  s = __builtin_fma(s, z, 1.0 / 362880);
  s = __builtin_fma(s, z, -1.0 / 5040);
  s = __builtin_fma(s, z, 1.0 / 120);
  s = __builtin_fma(s, z, -1.0 / 6);
  s = __builtin_fma(s, z, 1.0) * x;
  double c = -1.0 / 3628800;
  c = __builtin_fma(c, z, 1.0 / 40320);
  c = __builtin_fma(c, z, -1.0 / 720);
  c = __builtin_fma(c, z, 1.0 / 24);
  c = __builtin_fma(c, z, -0.5);
  c = __builtin_fma(c, z, 1.0);
  // By q quarters: (c, s), (-s, c), (-c, -s), (s, -c).
  const int q = (int)quarters & 3;
  const double cq = q & 1 ? s : c, sq = q & 1 ? c : s;
  return make_float2((float)((q == 1 || q == 2 ? -cq : cq) * magnitude),
                     (float)((q & 2 ? -sq : sq) * magnitude));
}

// float32 -> bf16 bits, to nearest even (v_cvt_pk_bf16_f32; a NaN stays one).
__device__ __forceinline__ uint32_t to_bf16(float v) { return __builtin_bit_cast(uint16_t, (__bf16)v); }

// The position of a token: int32 or int64.
__device__ __forceinline__ int64_t position_at(const void* positions, int wide, int64_t token) {
  return wide ? static_cast<const int64_t*>(positions)[token] : static_cast<const int32_t*>(positions)[token];
}

}  // namespace rotary_core
}  // namespace dsa
