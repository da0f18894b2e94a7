// Shared parts of the dense attention kernels (prompt_attention.hip,
// shared_prefix.hip): vector types, the matrix products of both 16-bit types,
// LDS access, and the join of partial results over split keys.
#pragma once

#include <type_traits>

#include "dsa_common.h"

namespace dsa {
namespace {

typedef __bf16 v8bf __attribute__((ext_vector_type(8)));
typedef __bf16 v2bf __attribute__((ext_vector_type(2)));
typedef _Float16 v8hf __attribute__((ext_vector_type(8)));
typedef _Float16 v2hf __attribute__((ext_vector_type(2)));
typedef float v2f __attribute__((ext_vector_type(2)));
typedef float v4f __attribute__((ext_vector_type(4)));
typedef float v16f __attribute__((ext_vector_type(16)));
typedef uint32_t v2u __attribute__((ext_vector_type(2)));
typedef uint32_t v4u __attribute__((ext_vector_type(4)));
typedef short v4s __attribute__((ext_vector_type(4)));
typedef v4s __attribute__((address_space(3))) * lds_v4s;

constexpr float kLog2E = 1.4426950408889634f;
// A row's running maximum is raised only when a block's exceeds it by more than
// this, in log2 units: probabilities stay at or below 2^(8 + kLift), and the
// accumulators are seldom rescaled.
constexpr float kLazyRescale = 8.0f;

// The 16-bit element type of a kernel: its matrix product over 16 dims of 32
// rows by 32 columns, and two floats rounded to nearest even into a pair. kLift: the
// log2 of the probability that a row's maximum has when it is raised.
struct Bf16 {
  static constexpr float kLift = 0.0f;
  static __device__ __forceinline__ v16f mfma(v4u a, v4u b, v16f c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(v8bf, a), __builtin_bit_cast(v8bf, b), c, 0, 0, 0);
  }
  static __device__ __forceinline__ uint32_t pack(float lo, float hi) {
    return __builtin_bit_cast(uint32_t, __builtin_convertvector((v2f){lo, hi}, v2bf));
  }
  // c plus both values of a pair, in fp32.
  static __device__ __forceinline__ float add_pair(uint32_t pair, float c) {
    return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(v2bf, pair), __builtin_bit_cast(v2bf, 0x3F803F80u), c, false);
  }
};
// fp16 holds 2^15 and loses bits below 2^-14: 2^7 at the maximum uses the range up to there,
// and what is lost lies 7 binades lower (with 1 at the maximum 60,000 keys of 2^-26 each,
// 9e-4 of the sum, went missing, and those of 2^-20 were off by up to 2^-6).
struct F16 {
  static constexpr float kLift = 7.0f;
  static __device__ __forceinline__ v16f mfma(v4u a, v4u b, v16f c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(v8hf, a), __builtin_bit_cast(v8hf, b), c, 0, 0, 0);
  }
  static __device__ __forceinline__ uint32_t pack(float lo, float hi) {
    return __builtin_bit_cast(uint32_t, __builtin_convertvector((v2f){lo, hi}, v2hf));
  }
  static __device__ __forceinline__ float add_pair(uint32_t pair, float c) {
    return __builtin_amdgcn_fdot2(__builtin_bit_cast(v2hf, pair), __builtin_bit_cast(v2hf, 0x3C003C00u), c, false);
  }
};

template <typename T>
__device__ __forceinline__ T lds_load(uint32_t addr) {
  return *(T __attribute__((address_space(3)))*)(uintptr_t)addr;
}
template <typename T>
__device__ __forceinline__ void lds_store(uint32_t addr, T v) {
  *(T __attribute__((address_space(3)))*)(uintptr_t)addr = v;
}

// Four 16-bit values of one column out of four rows: within 16 lanes, lane
// 4 r + q addresses 8 bytes (columns 4 q ..) of row r and lane c receives column c.
__device__ __forceinline__ v2u lds_column(uint32_t addr) {
  return __builtin_bit_cast(v2u, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s)(uintptr_t)addr));
}

// LDS barrier: this wave's LDS traffic done, then s_barrier; no memory access
// moves across it.
__device__ __forceinline__ void lds_barrier() {
  asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
}

template <int kOutstanding>
__device__ __forceinline__ void wait_loads() {
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(kOutstanding) : "memory");
}

// 16 bytes per lane from base + off + kFrom into LDS at lds_base + kTo + 16 * lane.
// (The instruction's offset counts on both sides.)
template <int kFrom, int kTo>
__device__ __forceinline__ void load_to_lds(const void* base, uint32_t off, uint32_t lds_base) {
  asm volatile("s_add_u32 m0, %0, %3\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2 offset:%4"
               ::"s"(lds_base), "v"(off), "s"(base), "n"(kTo - kFrom), "n"(kFrom) : "memory", "m0", "scc");
}

template <int kCount, int kAt = 0, typename F>
__device__ __forceinline__ void static_for(F f) {
  if constexpr (kAt < kCount) {
    f(std::integral_constant<int, kAt>{});
    static_for<kCount, kAt + 1>(f);
  }
}

// The larger of a value in lane l and lane l ^ 32, in both.
__device__ __forceinline__ float max_halves(float v) {
  const uint32_t u = __float_as_uint(v);
  const auto both = __builtin_amdgcn_permlane32_swap(u, u, false, false);
  return fmaxf(__uint_as_float(both[0]), __uint_as_float(both[1]));
}
__device__ __forceinline__ float sum_halves(float v) {
  const uint32_t u = __float_as_uint(v);
  const auto both = __builtin_amdgcn_permlane32_swap(u, u, false, false);
  return __uint_as_float(both[0]) + __uint_as_float(both[1]);
}

// A value's sum or largest over the wave, in every lane, by lane moves: xor 1 and 2 in
// a quad, the other quad of eight, the other eight, the other rows.
template <typename Op>
__device__ __forceinline__ uint32_t reduce_lanes(uint32_t v, Op op) {
  v = op(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0xB1, 0xF, 0xF, false));
  v = op(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x4E, 0xF, 0xF, false));
  v = op(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x141, 0xF, 0xF, false));
  v = op(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x140, 0xF, 0xF, false));
  const auto a = __builtin_amdgcn_permlane16_swap(v, v, false, false);
  v = op(a[0], a[1]);
  const auto b = __builtin_amdgcn_permlane32_swap(v, v, false, false);
  return op(b[0], b[1]);
}
__device__ __forceinline__ uint32_t sum_lanes(uint32_t v) {
  return reduce_lanes(v, [](uint32_t x, uint32_t y) { return x + y; });
}
__device__ __forceinline__ uint32_t max_lanes(uint32_t v) {
  return reduce_lanes(v, [](uint32_t x, uint32_t y) { return x > y ? x : y; });
}

// The sum over the lanes below this one: within rows of 16, then of the rows before.
__device__ __forceinline__ uint32_t sum_below(uint32_t v) {
  const uint32_t own = v;
  v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x111, 0xF, 0xF, true);
  v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x112, 0xF, 0xF, true);
  v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x114, 0xF, 0xF, true);
  v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x118, 0xF, 0xF, true);
  const uint32_t row = (threadIdx.x & 63) >> 4;
  const uint32_t r0 = __builtin_amdgcn_readlane((int)v, 15), r1 = __builtin_amdgcn_readlane((int)v, 31),
                 r2 = __builtin_amdgcn_readlane((int)v, 47);
  return v - own + (row > 0 ? r0 : 0) + (row > 1 ? r1 : 0) + (row > 2 ? r2 : 0);
}

// The running maximum, less the type's kLift, and sum of one row of scores (held by
// lanes l and l ^ 32: the maximum by both, of the sum a part each).
struct RowState {
  float top, sum;
};

// The maximum of a row's 32 scores, in log2 units (both halves).
__device__ __forceinline__ float row_max(const v16f& s, float scale_log2) {
  float mx = fmaxf(s[0], s[1]);
#pragma unroll
  for (int i = 2; i < 16; i += 2) mx = fmaxf(fmaxf(mx, s[i]), s[i + 1]);
  return max_halves(mx) * scale_log2;
}

// Whether a row's running maximum (-inf: no visible key so far) has to rise to take in
// scores up to mx. (Far from zero a score's own steps may exceed what fp16 has left above
// 2^15: there it rises earlier, from 2^24 on within 2^7 of the maximum.)
template <typename E>
__device__ __forceinline__ bool must_raise(const RowState& row, float mx) {
  const float most = row.top + (E::kLift + kLazyRescale);
  if constexpr (E::kLift > 0.0f) return mx > __builtin_fmaf(__builtin_fabsf(row.top), -0x1p-21f, most);
  return mx > most;
}

// Raises it; returns the factor for what was summed before (1 with no visible key so
// far: those sums are zeros, which are not worth a pass over the accumulators).
template <typename E>
__device__ __forceinline__ float raise(RowState& row, float mx) {
  if (!must_raise<E>(row, mx)) return 1.0f;
  const float top = fmaxf(row.top, mx - E::kLift);
  const float factor = row.top == -__builtin_inff() ? 1.0f : __builtin_amdgcn_exp2f(row.top - top);
  row.top = top;
  row.sum *= factor;
  return factor;
}

// A row's probabilities in log2 units against its running maximum, p = 2^(scale s +
// shift) with shift = -top (or 0 with no visible key so far: every score is then
// -inf and p = 0), as packed pairs whose rounded values join the row's sum. Issued
// in ticks of at most six instructions: tick t scales pair t, takes the powers of
// pair t - 1 and packs pair t - 2, so that none waits for the one before it.
template <typename E>
struct Softener {
  float x[2][2], y[2][2];
  template <typename Scores, typename Sum>
  __device__ __forceinline__ void tick(int t, int pairs, float scale_log2, Scores score, const float* shift, Sum put) {
    if (t >= 2) put(t - 2, E::pack(y[t & 1][0], y[t & 1][1]));
    if (t >= 1 && t - 1 < pairs) {
      y[(t - 1) & 1][0] = __builtin_amdgcn_exp2f(x[(t - 1) & 1][0]);
      y[(t - 1) & 1][1] = __builtin_amdgcn_exp2f(x[(t - 1) & 1][1]);
    }
    if (t < pairs) {
      x[t & 1][0] = __builtin_fmaf(score(2 * t), scale_log2, shift[t >> 3]);
      x[t & 1][1] = __builtin_fmaf(score(2 * t + 1), scale_log2, shift[t >> 3]);
    }
  }
};
__device__ __forceinline__ float shift_of(const RowState& row) {
  return row.top == -__builtin_inff() ? 0.0f : -row.top;
}

// A per-lane LDS address formed once and hidden from the optimizer, so that reads
// at constant distances use the instruction's offset field.
__device__ __forceinline__ uint32_t opaque(uint32_t v) {
  asm volatile("" : "+v"(v));
  return v;
}

// The value of lane J of a lane's quad (four neighbours).
template <int J>
__device__ __forceinline__ uint32_t quad_lane(uint32_t v) {
  return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, J * 0x55, 0xF, 0xF, true);
}

// x of the second of two lanes that kMove exchanges, and y of the first, trade places.
template <int kMove>
__device__ __forceinline__ void trade_lanes(uint32_t& x, uint32_t& y, bool second) {
  const uint32_t other_x = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, kMove, 0xF, 0xF, true);
  const uint32_t other_y = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)y, kMove, 0xF, 0xF, true);
  x = second ? other_y : x;
  y = second ? y : other_x;
}

// Vector j of lane i of each quad and vector i of its lane j trade places.
__device__ __forceinline__ void transpose_quad(v4u* w) {
  const bool odd = threadIdx.x & 1, high = threadIdx.x & 2;
  constexpr int kXor1 = 0xB1, kXor2 = 0x4E;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    uint32_t v[4] = {w[0][e], w[1][e], w[2][e], w[3][e]};
    trade_lanes<kXor1>(v[0], v[1], odd);
    trade_lanes<kXor1>(v[2], v[3], odd);
    trade_lanes<kXor2>(v[0], v[2], high);
    trade_lanes<kXor2>(v[1], v[3], high);
#pragma unroll
    for (int j = 0; j < 4; ++j) w[j][e] = v[j];
  }
}

// ------------------------------------------------- joining split keys --
// A row's keys may be split over work-groups: split s leaves its unscaled sum of
// p v (fp32 [splits][rows][dim]) and (maximum, sum of p) pairs ([splits][rows];
// split_stats). Their join is sum_s 2^(m_s - M) o_s / sum_s 2^(m_s - M) l_s.

// What a split leaves for a row: (-inf, 0) where nothing was visible (its values
// are then neither written nor read), a NaN maximum where a score was NaN.
__device__ __forceinline__ float2 split_stats(float top, float sum) {
  if (sum == 0.0f) return make_float2(-__builtin_inff(), 0.0f);
  return make_float2(sum == sum ? top : sum, sum);
}

// Joins them: kWays groups of kDim / 16 lanes take a row, 16 dims a lane (four
// vectors, each of neighbouring lanes side by side) and every kWays-th split each,
// against a running maximum of their own. What bounds it is reading the parts: many
// parts of few rows want many loads in flight.
template <typename E, int kDim, int kWays>
__global__ __launch_bounds__(kWays * kDim / 16 > 256 ? kWays * kDim / 16 : 256) void join_splits(
    const float* __restrict__ parts, const float2* __restrict__ stats, int64_t rows, int splits,
    const int32_t* __restrict__ cu, int32_t sequences, int64_t heads, uint16_t* __restrict__ out) {
  constexpr int kLanes = kDim / 16, kGroup = kWays * kLanes;
  constexpr int kThreads = kGroup > 256 ? kGroup : 256, kRows = kThreads / kGroup;
  __shared__ float shared[kRows][kWays][kDim];
  __shared__ float2 of_way[kRows][kWays];
  const int local = threadIdx.x / kGroup, way = threadIdx.x % kGroup / kLanes, l = threadIdx.x % kLanes;
  const int64_t row = (int64_t)blockIdx.x * kRows + local;
  const float none = -__builtin_inff();
  // Rows outside the sequences have no parts, and stay as they are.
  const bool live = row < rows && (cu == nullptr || (row >= cu[0] * heads && row < cu[sequences] * heads));
  if (live) {
    float4 acc[4] = {};
    float top = none, sum = 0.0f;
    constexpr int kAtOnce = 4;
    for (int s0 = way; s0 < splits; s0 += kWays * kAtOnce) {
      float2 st[kAtOnce];
      float4 o[kAtOnce][4];
#pragma unroll
      for (int i = 0; i < kAtOnce; ++i) {
        const int s = s0 + i * kWays;
        st[i] = s < splits ? stats[s * rows + row] : make_float2(none, 0.0f);
        // (A split without a visible key has written no values.)
        const float4* src = reinterpret_cast<const float4*>(parts + (s * rows + row) * kDim) + l;
        const bool some = st[i].y != 0.0f;
#pragma unroll
        for (int c = 0; c < 4; ++c) o[i][c] = some ? src[c * kLanes] : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      }
      float up = top;
#pragma unroll
      for (int i = 0; i < kAtOnce; ++i) up = fmaxf(up, st[i].x);
      const float keep = top == none ? 0.0f : __builtin_amdgcn_exp2f(top - up);
      sum *= keep;
#pragma unroll
      for (int c = 0; c < 4; ++c) acc[c].x *= keep, acc[c].y *= keep, acc[c].z *= keep, acc[c].w *= keep;
#pragma unroll
      for (int i = 0; i < kAtOnce; ++i) {
        // (A NaN maximum, of a split with a NaN score, spreads.)
        const float w = st[i].y != 0.0f ? __builtin_amdgcn_exp2f(st[i].x - up) : 0.0f;
        sum += w * st[i].y;
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          acc[c].x += w * o[i][c].x;
          acc[c].y += w * o[i][c].y;
          acc[c].z += w * o[i][c].z;
          acc[c].w += w * o[i][c].w;
        }
      }
      top = up;
    }
#pragma unroll
    for (int c = 0; c < 4; ++c) reinterpret_cast<float4*>(&shared[local][way][0])[c * kLanes + l] = acc[c];
    if (l == 0) of_way[local][way] = make_float2(top, sum);
  }
  __syncthreads();
  if (!live) return;
  float top = none;
#pragma unroll
  for (int w = 0; w < kWays; ++w) top = fmaxf(top, of_way[local][w].x);
  float sum = 0.0f, factor[kWays];
#pragma unroll
  for (int w = 0; w < kWays; ++w) {
    const float2 st = of_way[local][w];
    factor[w] = st.y != 0.0f ? (st.x == none ? st.y : __builtin_amdgcn_exp2f(st.x - top)) : 0.0f;
    sum += factor[w] * st.y;
  }
  const float inv = sum > 0.0f ? 1.0f / sum : (sum == 0.0f ? 0.0f : sum);
  for (int d = 2 * (threadIdx.x % kGroup); d < kDim; d += 2 * kGroup) {
    float a = 0.0f, b = 0.0f;
#pragma unroll
    for (int w = 0; w < kWays; ++w) {
      const float2 v = *reinterpret_cast<const float2*>(&shared[local][w][d]);
      a += factor[w] * v.x;
      b += factor[w] * v.y;
    }
    *reinterpret_cast<uint32_t*>(out + row * kDim + d) = E::pack(a * inv, b * inv);
  }
}

template <typename E, int kDim>
int launch_join(const float* parts, const float2* stats, int64_t rows, int splits, const int32_t* cu,
                int32_t sequences, int64_t heads, uint16_t* out, hipStream_t stream) {
  auto go = [&](auto kernel, int threads, int per_group) {
    hipLaunchKernelGGL(kernel, dim3((unsigned)((rows + per_group - 1) / per_group)), dim3(threads), 0, stream, parts,
                       stats, rows, splits, cu, sequences, heads, out);
  };
  // Ways for the parts there are.
  constexpr int kLanes = kDim / 16;
  if (splits <= 4) go(join_splits<E, kDim, 2>, 256, 256 / (2 * kLanes));
  else if (splits <= 32) go(join_splits<E, kDim, 8>, 256, 256 / (8 * kLanes));
  else go(join_splits<E, kDim, 32>, kLanes * 32 > 256 ? kLanes * 32 : 256, kLanes * 32 > 256 ? 1 : 256 / (32 * kLanes));
  DSA_CHECK_LAUNCH("join of split keys");
  return kOk;
}

}  // namespace
}  // namespace dsa
