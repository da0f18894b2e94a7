// Rotary positions of queries and keys: for pair i of a head's rotated part,
// t = position * frequency[i],
//   a' = m (a cos t - b sin t), b' = m (b cos t + a sin t)
// in fp32, rounded once to the element type; pairs (2 i, 2 i + 1) (interleaved)
// or (i, i + r / 2) (half); inverse: -t, the transposed map. Other dims of the
// head are copied (or left, in place).
//
// Bound by memory: each value is read and written once. A work-group takes some
// tokens (or a part of one token's heads) in items of eight pairs, two 16-byte
// vectors of 16-bit values, one per thread (two or four of them were no faster in
// 8,192 tokens of 128 heads, 55 us or 4.9 TB/s, and slower in small calls: 1,023
// fp32 tokens 17.1 us, with four 20.0); while they are on their way it forms the
// tokens' cosines and sines in LDS (64 bits, once for all heads; 16 tokens 6.6
// -> 3.4 us against forming them first).
// Types, offsets or strides that do not allow vectors take one pair at a time.
#include "rotary_core.h"
#include "../../include/dsa_gfx950.h"

namespace dsa {
namespace {

constexpr int kThreads = 256;
constexpr int kTableEntries = 2048;    // (cos, sin) of a work-group

struct RopeSide {
  const void* in;
  void* out;
  int64_t in_token, in_head, out_token, out_head;  // strides, elements
  int32_t heads;
  int32_t tokens_per_group, groups_per_token;      // one of them is 1
  int64_t groups;
};

struct RopeArgs {
  RopeSide side[2];
  const void* positions;
  const float* frequencies;
  int64_t tokens;
  int32_t wide_positions, dim, offset, half, interleaved, copy;
  double magnitude;
  float sign;
};

template <typename T>
__device__ __forceinline__ float to_f32(T v) { return (float)v; }
template <>
__device__ __forceinline__ float to_f32(uint16_t v) { return bf16_to_f32(v); }
template <typename T>
__device__ __forceinline__ T from_f32(float v) { return (T)v; }
template <>
__device__ __forceinline__ uint16_t from_f32(float v) { return (uint16_t)rotary_core::to_bf16(v); }

// A vector of 8 elements, aligned to 16 bytes.
template <typename T>
struct __align__(16) Eight {
  T v[8];
};

// T: uint16_t (bf16 bits), _Float16 or float. kVector: items of 8 pairs (or 16
// copied values), else of one.
template <typename T, bool kVector>
__global__ __launch_bounds__(kThreads) void rope_pair(const RopeArgs a) {
  __shared__ float2 table[kTableEntries];
  const bool second = (int64_t)blockIdx.x >= a.side[0].groups;
  const RopeSide& side = a.side[second];
  const int64_t group = blockIdx.x - (second ? a.side[0].groups : 0);
  const int64_t token0 = group / side.groups_per_token * side.tokens_per_group;
  const int tokens = (int)min((int64_t)side.tokens_per_group, a.tokens - token0);
  constexpr int kPairs = kVector ? 8 : 1;
  constexpr int kSpan = kVector ? 8 : 1;
  const int turned = a.half / kPairs;                              // items that rotate, per head
  const int copied = a.copy ? (a.dim - 2 * a.half) / (2 * kSpan) : 0;
  const int per_head = turned + copied;
  const int per_token = side.heads * per_head;
  // A part of one token's items, or all items of some tokens.
  const int part = (int)(group % side.groups_per_token);
  const int begin = part * kThreads;
  const int end = side.groups_per_token > 1 ? min(begin + kThreads, per_token) : tokens * per_token;
  const int item = begin + (int)threadIdx.x;
  const bool mine = item < end;
  T x[2 * kSpan];
  T *to0 = nullptr, *to1 = nullptr;
  int pair = -1;  // table entry of the item's first pair, -1: copied
  if (mine) {
    const int t = side.groups_per_token > 1 ? 0 : item / per_token;
    const int rest = item - t * per_token;
    const int head = rest / per_head, unit = rest - head * per_head;
    int at0, at1;  // the two vectors' dims
    if (unit < turned) {
      pair = t * a.half + unit * kPairs;
      at0 = a.offset + (a.interleaved ? 2 * unit * kSpan : unit * kSpan);
      at1 = at0 + (a.interleaved ? kSpan : a.half);
    } else {
      at0 = (unit - turned) * 2 * kSpan;
      at1 = at0 + kSpan;
      if (at0 >= a.offset) at0 += 2 * a.half;
      if (at1 >= a.offset) at1 += 2 * a.half;
    }
    const T* in = static_cast<const T*>(side.in) + (token0 + t) * side.in_token + head * side.in_head;
    T* out = static_cast<T*>(side.out) + (token0 + t) * side.out_token + head * side.out_head;
    to0 = out + at0;
    to1 = out + at1;
    if constexpr (kVector) {
      *reinterpret_cast<Eight<T>*>(&x[0]) = *reinterpret_cast<const Eight<T>*>(in + at0);
      *reinterpret_cast<Eight<T>*>(&x[kSpan]) = *reinterpret_cast<const Eight<T>*>(in + at1);
    } else {
      x[0] = in[at0];
      x[1] = in[at1];
    }
  }
  for (int e = threadIdx.x; e < tokens * a.half; e += kThreads) {
    const int t = e / a.half;
    float2 cs = rotary_core::turn(rotary_core::position_at(a.positions, a.wide_positions, token0 + t),
                                  a.frequencies[e - t * a.half], a.magnitude);
    cs.y *= a.sign;
    table[e] = cs;
  }
  __syncthreads();
  if (!mine) return;
  if (pair >= 0) {
#pragma unroll
    for (int p = 0; p < kPairs; ++p) {
      const float2 cs = table[pair + p];
      T& xa = a.interleaved ? x[2 * p] : x[p];
      T& xb = a.interleaved ? x[2 * p + 1] : x[kSpan + p];
      const float u = to_f32(xa), v = to_f32(xb);
      xa = from_f32<T>(u * cs.x - v * cs.y);
      xb = from_f32<T>(v * cs.x + u * cs.y);
    }
  }
  if constexpr (kVector) {
    *reinterpret_cast<Eight<T>*>(to0) = *reinterpret_cast<Eight<T>*>(&x[0]);
    *reinterpret_cast<Eight<T>*>(to1) = *reinterpret_cast<Eight<T>*>(&x[kSpan]);
  } else {
    *to0 = x[0];
    *to1 = x[1];
  }
}

int64_t items_per_head(const RopeArgs& a, bool vector) {
  return vector ? a.half / 8 + (a.copy ? (a.dim - 2 * a.half) / 16 : 0)
                : a.half + (a.copy ? (a.dim - 2 * a.half) / 2 : 0);
}

template <typename T, bool kVector>
int launch_items(RopeArgs a, hipStream_t stream) {
  const int64_t per_head = items_per_head(a, kVector);
  int64_t groups = 0;
  for (RopeSide& s : a.side) {
    const int64_t per_token = per_head * s.heads;
    s.tokens_per_group = s.groups_per_token = 1;
    s.groups = 0;
    if (per_token == 0) continue;
    if (per_token >= kThreads) {
      s.groups_per_token = (int32_t)((per_token + kThreads - 1) / kThreads);
    } else {
      int64_t t = kThreads / per_token;
      if (t * a.half > kTableEntries) t = kTableEntries / a.half;
      s.tokens_per_group = (int32_t)t;
    }
    s.groups = (a.tokens + s.tokens_per_group - 1) / s.tokens_per_group * s.groups_per_token;
    groups += s.groups;
  }
  DSA_CHECK_ARG(grid_fits(groups, kThreads), "too many tokens for one launch");
  if (groups == 0) return kOk;
  hipLaunchKernelGGL((rope_pair<T, kVector>), dim3((unsigned)groups), dim3(kThreads), 0, stream, a);
  DSA_CHECK_LAUNCH("rope");
  return kOk;
}

template <typename T>
int launch_rope(const RopeArgs& a, bool vector, hipStream_t stream) {
  return vector ? launch_items<T, true>(a, stream) : launch_items<T, false>(a, stream);
}

}  // namespace
}  // namespace dsa

extern "C" int dsa_rope_pair(const void* q, int64_t q_token_stride, int64_t q_head_stride, void* q_out,
                             int64_t q_out_token_stride, int64_t q_out_head_stride, int64_t q_heads, const void* k,
                             int64_t k_token_stride, int64_t k_head_stride, void* k_out,
                             int64_t k_out_token_stride, int64_t k_out_head_stride, int64_t k_heads, int dtype,
                             int64_t tokens, int64_t dim, int64_t offset, int64_t rotated, const void* positions,
                             int wide_positions, const float* frequencies, double magnitude, int interleaved,
                             int inverse, hipStream_t stream) {
  using namespace dsa;
  DSA_CHECK_ARG(dtype >= 0 && dtype <= 2, "unknown element type");
  DSA_CHECK_ARG(tokens >= 0 && dim >= 1 && dim <= 65536 && q_heads >= 0 && k_heads >= 0 && q_heads <= 65536 &&
                    k_heads <= 65536 && q_heads * dim < (1 << 28) && k_heads * dim < (1 << 28),
                "invalid rope shape");
  DSA_CHECK_ARG(rotated >= 2 && rotated % 2 == 0 && rotated <= 2 * kTableEntries && offset >= 0 &&
                    offset + rotated <= dim && (dim - rotated) % 2 == 0,
                "the rotated part must be an even number of dims within the head, the rest even too");
  DSA_CHECK_ARG(__builtin_isfinite((float)magnitude), "magnitude must be finite");
  if (tokens == 0 || q_heads + k_heads == 0) return kOk;
  DSA_CHECK_ARG((q_heads == 0 || (q && q_out)) && (k_heads == 0 || (k && k_out)) && positions && frequencies,
                "null pointer");
  RopeArgs a{};
  a.side[0] = RopeSide{q, q_out, q_token_stride, q_head_stride, q_out_token_stride, q_out_head_stride,
                       (int32_t)q_heads, 1, 1, 0};
  a.side[1] = RopeSide{k, k_out, k_token_stride, k_head_stride, k_out_token_stride, k_out_head_stride,
                       (int32_t)k_heads, 1, 1, 0};
  a.positions = positions;
  a.frequencies = frequencies;
  a.tokens = tokens;
  a.wide_positions = wide_positions != 0;
  a.dim = (int32_t)dim, a.offset = (int32_t)offset, a.half = (int32_t)(rotated / 2);
  a.interleaved = interleaved != 0;
  a.magnitude = magnitude, a.sign = inverse ? -1.0f : 1.0f;
  // In place, what is not rotated stays where it is.
  auto in_place = [](const RopeSide& s) {
    return s.heads == 0 || (s.in == s.out && s.in_token == s.out_token && s.in_head == s.out_head);
  };
  a.copy = !(in_place(a.side[0]) && in_place(a.side[1]));
  // Vectors of 8 elements where every one of them is aligned (fp32: to 16 of its
  // 32 bytes).
  bool vector = rotated % 16 == 0 && offset % 8 == 0 && (dim - rotated) % 16 == 0;
  const int64_t size = dtype == DSA_DTYPE_F32 ? 4 : 2, align = 16 / size;
  for (const RopeSide& s : a.side) {
    if (s.heads == 0) continue;
    vector = vector && reinterpret_cast<uintptr_t>(s.in) % 16 == 0 && reinterpret_cast<uintptr_t>(s.out) % 16 == 0;
    for (int64_t stride : {s.in_token, s.in_head, s.out_token, s.out_head}) vector = vector && stride % align == 0;
  }
  if (dtype == DSA_DTYPE_BF16) return launch_rope<uint16_t>(a, vector, stream);
  if (dtype == DSA_DTYPE_F16) return launch_rope<_Float16>(a, vector, stream);
  return launch_rope<float>(a, vector, stream);
}
