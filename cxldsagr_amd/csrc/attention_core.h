// Shared parts of the dense attention kernels (prompt_attention.hip,
// shared_prefix.hip): vector types, the matrix products of both 16-bit types,
// LDS access, and the join of partial results over split keys.
#pragma once

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
// this, in log2 units: probabilities stay at or below 2^8 (exact in range for
// both 16-bit types), and the accumulators are seldom rescaled.
constexpr float kLazyRescale = 8.0f;

// The 16-bit element type of a kernel: its matrix product over 16 dims of 32
// rows by 32 columns, and two floats rounded to nearest even into a pair.
struct Bf16 {
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
struct F16 {
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

// 16 bytes per lane from base + off into LDS at lds_base + 16 * lane.
__device__ __forceinline__ void load_to_lds(const void* base, uint32_t off, uint32_t lds_base) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2"
               ::"s"(lds_base), "v"(off), "s"(base) : "memory", "m0");
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

// The running maximum and sum of one row of scores (held by lanes l and l ^ 32:
// the maximum by both, of the sum a part each).
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

// Whether a row's running maximum has to rise to take in scores up to mx.
__device__ __forceinline__ bool must_raise(const RowState& row, float mx) {
  const float none = -__builtin_inff();
  return mx > row.top + kLazyRescale || (row.top == none && mx != none);
}

// Raises it; returns the factor for what was summed before.
__device__ __forceinline__ float raise(RowState& row, float mx) {
  if (!must_raise(row, mx)) return 1.0f;
  const float top = fmaxf(row.top, mx);
  const float factor = __builtin_amdgcn_exp2f(row.top - top);
  row.top = top;
  row.sum *= factor;
  return factor;
}

// One pair of probabilities, in log2 units against the row's running maximum
// (shift = -top, or 0 with no visible key so far: every score is then -inf and
// p = 0); the rounded values join the row's sum.
template <typename E>
__device__ __forceinline__ uint32_t probability_pair(float s0, float s1, float scale_log2, float shift, float& sum) {
  const uint32_t p = E::pack(__builtin_amdgcn_exp2f(__builtin_fmaf(s0, scale_log2, shift)),
                             __builtin_amdgcn_exp2f(__builtin_fmaf(s1, scale_log2, shift)));
  sum = E::add_pair(p, sum);
  return p;
}
__device__ __forceinline__ float shift_of(const RowState& row) {
  return row.top == -__builtin_inff() ? 0.0f : -row.top;
}

// A per-lane LDS address formed once and hidden from the optimizer (an identity
// lane move), so that reads at constant distances use the instruction's offset.
__device__ __forceinline__ uint32_t opaque_address(uint32_t v) {
  return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0xE4, 0xF, 0xF, false);
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

// Joins them: four groups of kDim / 8 lanes take a row, a quarter of its splits
// each, 8 dims a lane. What bounds it is reading the parts.
template <typename E, int kDim>
__global__ __launch_bounds__(256) void join_splits(const float* __restrict__ parts, const float2* __restrict__ stats,
                                                   int64_t rows, int splits, const int32_t* __restrict__ cu,
                                                   int32_t sequences, int64_t heads, uint16_t* __restrict__ out) {
  constexpr int kLanes = kDim / 8, kWays = 4, kRows = 256 / (kLanes * kWays);
  __shared__ float shared[kWays][kRows][kDim + 4];
  const int local = threadIdx.x / (kLanes * kWays);
  const int way = threadIdx.x / kLanes % kWays;
  const int d = (threadIdx.x % kLanes) * 8;
  const int64_t row = (int64_t)blockIdx.x * kRows + local;
  // Rows outside the sequences have no parts, and stay as they are.
  const bool live = row < rows && (cu == nullptr || (row >= cu[0] * heads && row < cu[sequences] * heads));
  float acc[8] = {}, sum = 0.0f;
  if (live) {
    float top = -__builtin_inff();
    for (int s = 0; s < splits; ++s) top = fmaxf(top, stats[s * rows + row].x);
#pragma unroll 4
    for (int s = way; s < splits; s += kWays) {
      const float2 st = stats[s * rows + row];
      if (st.x == -__builtin_inff()) continue;  // (a NaN maximum, of a split with NaN scores, spreads)
      const float w = __builtin_amdgcn_exp2f(st.x - top);
      sum += w * st.y;
      const float4* o = reinterpret_cast<const float4*>(parts + (s * rows + row) * kDim + d);
      const float4 a = o[0], b = o[1];
      acc[0] += w * a.x, acc[1] += w * a.y, acc[2] += w * a.z, acc[3] += w * a.w;
      acc[4] += w * b.x, acc[5] += w * b.y, acc[6] += w * b.z, acc[7] += w * b.w;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) shared[way][local][d + i] = acc[i];
    if (d == 0) shared[way][local][kDim] = sum;
  }
  __syncthreads();
  if (!live || way != 0) return;
#pragma unroll
  for (int w = 1; w < kWays; ++w) {
    sum = w == 1 ? shared[0][local][kDim] + shared[w][local][kDim] : sum + shared[w][local][kDim];
#pragma unroll
    for (int i = 0; i < 8; ++i) acc[i] += shared[w][local][d + i];
  }
  const float inv = sum > 0.0f ? 1.0f / sum : (sum == 0.0f ? 0.0f : sum);
  v4u packed;
#pragma unroll
  for (int i = 0; i < 4; ++i) packed[i] = E::pack(acc[2 * i] * inv, acc[2 * i + 1] * inv);
  *reinterpret_cast<v4u*>(out + row * kDim + d) = packed;
}

template <typename E, int kDim>
int launch_join(const float* parts, const float2* stats, int64_t rows, int splits, const int32_t* cu,
                int32_t sequences, int64_t heads, uint16_t* out, hipStream_t stream) {
  constexpr int kRows = 256 / (kDim / 8 * 4);
  hipLaunchKernelGGL((join_splits<E, kDim>), dim3((unsigned)((rows + kRows - 1) / kRows)), dim3(256), 0, stream, parts,
                     stats, rows, splits, cu, sequences, heads, out);
  DSA_CHECK_LAUNCH("join of split keys");
  return kOk;
}

}  // namespace
}  // namespace dsa
