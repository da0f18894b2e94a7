// Each token's experts from its logits:
//   s = sigmoid(l) or softmax(l), rounded to 32 bits;  b = s + bias (32 bits);
//   of each group of experts the best b, with a bias the sum of its two best (32 bits);
//   the k largest b of the top_groups best groups, in that order, ties to the lower index;
//   w = s, or s / (their sum + 1e-20), times scale, rounded once to 32 bits.
// Scores are formed in 64 bits and rounded once, so that the order is that of the definition
// and not of some exponential's last bits. A NaN is larger than every number (as in a sort),
// so that it shows in the weights.
//
// kLanes lanes take a token, some lanes a group: a group's experts are cut into runs of
// `per`, one for each of `parts` lanes (a power of two), so that every count of experts and
// groups fits. An expert's rank is one number of 43 bits, its b as an ordered integer above
// its slot counted down (slots are in the experts' order), held as a positive double of those
// bits: v_max_f64 compares them in one instruction, and no two are equal. k times the largest
// is found over the lanes and struck out.
#include "attention_core.h"
#include "../../include/dsa_gfx950.h"

namespace dsa {
namespace {

constexpr int kThreads = 256;
constexpr int kMaxExperts = 1024, kMaxGroups = 64, kMaxChoices = 64;

struct RouteArgs {
  const void* logits;
  const float* bias;  // or null
  float* weights;
  int32_t* ids;
  int64_t stride, tokens;
  int32_t k, groups, top_groups, size, parts, log_parts, per, softmax, renormalize, vectors;
  double scale;
};

__device__ __forceinline__ float value_of(uint16_t v) { return bf16_to_f32(v); }
__device__ __forceinline__ float value_of(_Float16 v) { return (float)v; }
__device__ __forceinline__ float value_of(float v) { return v; }

// Floats as integers of the same order; NaN above all. (0 is below -inf's.)
__device__ __forceinline__ uint32_t ordered(float v) {
  const uint32_t b = __float_as_uint(v);
  return v != v ? 0xFFFFFFFFu : (b >> 31 ? ~b : b | 0x80000000u);
}
__device__ __forceinline__ float from_ordered(uint32_t k) {
  return __uint_as_float(k == 0xFFFFFFFFu ? kCanonicalNan : (k >> 31 ? k & 0x7FFFFFFFu : ~k));
}

// A value's exchange over the lanes of a token, in rows of 16 and then between them: step i
// hands every lane that of one whose first 2^i neighbours are the others' (lanes that
// differ in bit 0, in bit 1, then mirrored within 8 and 16, then in bits 4 and 5).
template <int kStep>
__device__ __forceinline__ uint32_t neighbour(uint32_t v) {
  if constexpr (kStep < 4) {
    constexpr int kMoves[4] = {0xB1, 0x4E, 0x141, 0x140};
    return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, kMoves[kStep], 0xF, 0xF, false);
  } else if constexpr (kStep == 4) {
    const auto both = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    return (threadIdx.x & 16) ? both[0] : both[1];
  } else {
    const auto both = __builtin_amdgcn_permlane32_swap(v, v, false, false);
    return (threadIdx.x & 32) ? both[0] : both[1];
  }
}
template <int kLanes, typename Op>
__device__ __forceinline__ double over_lanes(double v, Op op) {
  static_for<kLanes == 64 ? 6 : 4>([&](auto step) {
    const uint64_t b = __builtin_bit_cast(uint64_t, v);
    const uint32_t lo = neighbour<decltype(step)::value>((uint32_t)b), hi = neighbour<decltype(step)::value>((uint32_t)(b >> 32));
    v = op(v, __builtin_bit_cast(double, (uint64_t)hi << 32 | lo));
  });
  return v;
}

// The larger of two positive numbers. (Not fmax, which has each first made a quiet NaN if
// it were a signalling one.)
__device__ __forceinline__ double larger(double x, double y) {
  double v;
  asm("v_max_f64 %0, %1, %2" : "=v"(v) : "v"(x), "v"(y));
  return v;
}

// e^z to 2^-46 for z of at most 110 in magnitude: 2^n times the power series of the rest,
// within 0.35 of 0, up to the 11th power. near: z in 32 bits, for n alone.
__device__ __forceinline__ double exponential(double z, float near) {
  const float n = __builtin_rintf(near * kLog2E);
  // ln 2 as 32 bits (so that n times them is exact) and what is left.
  double r = __builtin_fma((double)n, -0x1.62e42fee00000p-1, z);
  r = __builtin_fma((double)n, -0x1.a39ef35793c76p-33, r);
  double p = 1.0 / 39916800.0;
  constexpr double kTerms[] = {1.0 / 3628800.0, 1.0 / 362880.0, 1.0 / 40320.0, 1.0 / 5040.0, 1.0 / 720.0, 1.0 / 120.0,
                               1.0 / 24.0, 1.0 / 6.0, 0.5, 1.0, 1.0};
#pragma unroll
  for (double term : kTerms) p = __builtin_fma(p, r, term);
  // (p is between 0.7 and 1.5, n at most 159: its exponent has room.)
  const uint64_t bits = __builtin_bit_cast(uint64_t, p);
  const uint32_t high = (uint32_t)(bits >> 32) + ((uint32_t)(int32_t)n << 20);
  return __builtin_bit_cast(double, (uint64_t)high << 32 | (uint32_t)bits);
}

// 1 / v for v of normal size, to 2^-46: the unit's estimate and a step.
__device__ __forceinline__ double reciprocal(double v) {
  const double y = __builtin_amdgcn_rcp(v);
  return __builtin_fma(__builtin_fma(-v, y, 1.0), y, y);
}

// A score of 32 bits is 0 below an exponent of -104 and does not feel a sum's e^-104 beside
// 1: exponents are cut off there, at this.
constexpr float kFar = 110.0f;

// kSlots neighbours from `from` on, of which `end` are there: as vectors where every lane's
// are whole and aligned, else one by one (past the end the last again).
template <typename T, int kSlots>
__device__ __forceinline__ void load_slots(float (&to)[kSlots], const T* from, int end, bool vectors) {
  constexpr int kFew = 16 / sizeof(T);
  if (kSlots % kFew == 0 && vectors) {
    struct __align__(16) Few {
      T v[kFew];
    };
#pragma unroll
    for (int i = 0; i + kFew <= kSlots; i += kFew) {
      const Few few = *reinterpret_cast<const Few*>(from + i);
#pragma unroll
      for (int j = 0; j < kFew; ++j) to[i + j] = value_of(few.v[j]);
    }
    return;
  }
#pragma unroll
  for (int i = 0; i < kSlots; ++i) to[i] = value_of(from[i < end ? i : end - 1]);
}

template <typename T, int kLanes, int kSlots>
__global__ __launch_bounds__(kThreads) void route(RouteArgs a) {
  constexpr int kTokens = kThreads / kLanes;
  __shared__ float scores[kTokens][kLanes * kSlots + kTokens];  // (a lane's slots side by side)
  __shared__ uint32_t of_group[kTokens][kMaxGroups];
  __shared__ int32_t chosen[kTokens][kMaxChoices];
  const int l = threadIdx.x % kLanes, local = threadIdx.x / kLanes;
  const int64_t own = (int64_t)blockIdx.x * kTokens + local;
  const bool live = own < a.tokens;
  const T* logits = static_cast<const T*>(a.logits) + (live ? own : a.tokens - 1) * a.stride;
  const int group = l >> a.log_parts, from = (l & (a.parts - 1)) * a.per;
  const int end = group < a.groups ? (a.size - from < a.per ? a.size - from : a.per) : 0;  // this lane's slots
  const int first = end > 0 ? group * a.size + from : 0;

  float s[kSlots], bias[kSlots];
  load_slots<T, kSlots>(s, logits + first, end > 0 ? end : 1, a.vectors & 1);
  if (a.bias) {
    load_slots<float, kSlots>(bias, a.bias + first, end > 0 ? end : 1, a.vectors & 2);
  } else {
#pragma unroll
    for (int i = 0; i < kSlots; ++i) bias[i] = 0.0f;  // (A score is not below 0: this adds nothing.)
  }
  // (NaN: its score is one, added so that no branch goes round the others' work.)
  float nan[kSlots];
#pragma unroll
  for (int i = 0; i < kSlots; ++i) nan[i] = s[i] == s[i] ? 0.0f : s[i];
  if (a.softmax) {
    float top = s[0];
#pragma unroll
    for (int i = 1; i < kSlots; ++i) top = fmaxf(top, s[i]);
    if (end <= 0) top = -__builtin_inff();
    const double most = over_lanes<kLanes>((double)top, [](double x, double y) { return __builtin_fmax(x, y); });
    // (A row's infinity, or nothing but its opposite, makes NaN of all, as the quotient.)
    const double nothing = most - most;
    double e[kSlots], sum = 0.0;
#pragma unroll
    for (int i = 0; i < kSlots; ++i) {
      const double z = __builtin_fmax((double)s[i] - most, (double)-kFar);
      e[i] = exponential(z, (float)z) + (double)nan[i];
      sum += i < end ? e[i] : 0.0;
    }
    sum = reciprocal(over_lanes<kLanes>(sum + nothing, [](double x, double y) { return x + y; }));
#pragma unroll
    for (int i = 0; i < kSlots; ++i) s[i] = (float)(e[i] * sum);
  } else {
#pragma unroll
    for (int i = 0; i < kSlots; ++i) {
      const float z = __builtin_amdgcn_fmed3f(-s[i], -kFar, kFar);
      s[i] = (float)reciprocal(1.0 + exponential(z, z)) + nan[i];
    }
  }

#pragma unroll
  for (int i = 0; i < kSlots; ++i) scores[local][l * kSlots + i] = s[i];
  uint32_t key[kSlots];
#pragma unroll
  for (int i = 0; i < kSlots; ++i) key[i] = ordered(s[i] + bias[i]) & (i < end ? ~0u : 0u);
  if (a.top_groups < a.groups) {
    uint32_t one = 0, two = 0;  // the group's best and next
#pragma unroll
    for (int i = 0; i < kSlots; ++i) {
      const uint32_t less = min(key[i], one);
      one = max(key[i], one);
      two = max(two, less);
    }
    static_for<kLanes == 64 ? 6 : 4>([&](auto step) {
      if (a.log_parts <= decltype(step)::value) return;
      const uint32_t o1 = neighbour<decltype(step)::value>(one), o2 = neighbour<decltype(step)::value>(two);
      two = max(min(one, o1), max(two, o2));
      one = max(one, o1);
    });
    const uint32_t mine = a.bias && two ? ordered(from_ordered(one) + from_ordered(two)) : one;
    if ((l & (a.parts - 1)) == 0) of_group[local][group] = mine;
    __syncthreads();
    int better = 0;
    for (int g = 0; g < a.groups; ++g) {
      const uint32_t other = of_group[local][g];
      better += (other > mine) | ((other == mine) & (g < group));
    }
#pragma unroll
    for (int i = 0; i < kSlots; ++i) key[i] = better < a.top_groups ? key[i] : 0u;
  }

  // (What is not eligible keeps a rank below all that are.)
  uint32_t high[kSlots], low[kSlots];
#pragma unroll
  for (int i = 0; i < kSlots; ++i) {
    high[i] = key[i] >> 2;
    low[i] = key[i] << 30 | (uint32_t)(2047 - (l * kSlots + i)) << 19;
  }
  auto rank = [&](int i) { return __builtin_bit_cast(double, (uint64_t)high[i] << 32 | low[i]); };
  for (int c = 0; c < a.k; ++c) {
    double best = rank(0);
#pragma unroll
    for (int i = 1; i < kSlots; ++i) best = larger(best, rank(i));
    best = over_lanes<kLanes>(best, larger);
#pragma unroll
    for (int i = 0; i < kSlots; ++i) high[i] = rank(i) == best ? 0u : high[i];
    if (l == 0) chosen[local][c] = 2047 - (int32_t)(__builtin_bit_cast(uint64_t, best) >> 19 & 2047);
  }
  __syncthreads();
  if (!live) return;
  // (In 64 bits up to the weight's own rounding: in 32 the sum, the quotient and the product each
  // added theirs.)
  double factor = a.scale;
  if (a.renormalize) {
    double sum = 1e-20;
    for (int c = 0; c < a.k; ++c) sum += (double)scores[local][chosen[local][c]];
    factor *= reciprocal(sum);
  }
  for (int c = l; c < a.k; c += kLanes) {
    const int at = chosen[local][c], lane = at / kSlots;
    a.weights[own * a.k + c] = (float)((double)scores[local][at] * factor);
    a.ids[own * a.k + c] = (lane >> a.log_parts) * a.size + (lane & (a.parts - 1)) * a.per + at % kSlots;
  }
}

template <typename T>
int launch_route(RouteArgs a, hipStream_t stream) {
  // Lanes of a token, of a group, and a lane's experts.
  auto plan = [&](int lanes) {
    a.log_parts = 0;
    while (2 * a.groups << a.log_parts <= lanes) ++a.log_parts;
    a.parts = 1 << a.log_parts;
    a.per = (a.size + a.parts - 1) / a.parts;
  };
  auto go = [&](auto kernel, int lanes, int slots) {
    const int64_t tokens = kThreads / lanes, few = 16 / sizeof(T);
    const bool whole = a.per == slots && a.per * a.parts == a.size && a.parts * a.groups == lanes;
    auto aligned = [](const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; };
    a.vectors = (whole && slots % few == 0 && a.stride % few == 0 && aligned(a.logits) ? 1 : 0) |
                (whole && slots % 4 == 0 && aligned(a.bias) ? 2 : 0);
    hipLaunchKernelGGL(kernel, dim3((unsigned)((a.tokens + tokens - 1) / tokens)), dim3(kThreads), 0, stream, a);
  };
  // Four tokens a wave share the lanes' exchanges, half the instructions per token; with few
  // tokens a whole wave for one ends sooner (a wave for one against four a wave: 256 experts 3,000
  // tokens 6.2 us against 6.8, 4,096 7.2 against 6.8; 160 experts 2,048 5.4 against 5.8, 2,560 6.2
  // against 5.8; 128 experts 1,024 3.9 against 4.3, 2,048 4.5 against 4.3; 64 experts 1,024 3.5
  // against 3.4). A lane's slots come by fours, whole loads of 32 bits: with 16 for all beyond 8,
  // 16,384 tokens of 160 experts took 13.2 us (10.6 with 12), of 192 12.7 (9.8), of 144 12.6 (10.4).
  plan(16);
  if (a.tokens >= 256 * a.per && a.groups <= 16 && a.per <= 16) {
    if (a.per <= 4) go(route<T, 16, 4>, 16, 4);
    else if (a.per <= 8) go(route<T, 16, 8>, 16, 8);
    else if (a.per <= 12) go(route<T, 16, 12>, 16, 12);
    else go(route<T, 16, 16>, 16, 16);
    DSA_CHECK_LAUNCH("routing to experts");
    return kOk;
  }
  plan(64);
  if (a.per <= 2) go(route<T, 64, 2>, 64, 2);
  else if (a.per <= 4) go(route<T, 64, 4>, 64, 4);
  else if (a.per <= 16) go(route<T, 64, 16>, 64, 16);
  else go(route<T, 64, 32>, 64, 32);
  DSA_CHECK_LAUNCH("routing to experts");
  return kOk;
}

}  // namespace
}  // namespace dsa

extern "C" int dsa_route_experts(const void* logits, int64_t stride, int dtype, int64_t tokens, int64_t experts,
                                 int64_t k, const float* bias, int softmax, int64_t groups, int64_t top_groups,
                                 int renormalize, double scale, float* weights, int32_t* ids, hipStream_t stream) {
  using namespace dsa;
  DSA_CHECK_ARG(dtype >= 0 && dtype <= 2, "unknown element type");
  DSA_CHECK_ARG(tokens >= 0 && experts >= 1 && experts <= kMaxExperts, "experts must number 1 to %d", kMaxExperts);
  DSA_CHECK_ARG(groups >= 1 && groups <= kMaxGroups && experts % groups == 0 && top_groups >= 1 && top_groups <= groups,
                "groups must divide the experts and be at least top_groups, %d at most", kMaxGroups);
  DSA_CHECK_ARG(k >= 1 && k <= kMaxChoices && k <= top_groups * (experts / groups),
                "k must be 1 to %d and within the experts of top_groups groups", kMaxChoices);
  DSA_CHECK_ARG(__builtin_isfinite((float)scale), "scale must be finite");
  DSA_CHECK_ARG(tokens <= (1ll << 40) && grid_fits((tokens + 3) / 4, kThreads), "too many tokens for one launch");
  if (tokens == 0) return kOk;
  DSA_CHECK_ARG(logits && weights && ids, "null pointer");
  RouteArgs a{};
  a.logits = logits, a.bias = bias, a.weights = weights, a.ids = ids;
  a.stride = stride, a.tokens = tokens, a.k = (int32_t)k;
  a.groups = (int32_t)groups, a.top_groups = (int32_t)top_groups, a.size = (int32_t)(experts / groups);
  a.softmax = softmax != 0, a.renormalize = renormalize != 0, a.scale = scale;
  if (dtype == DSA_DTYPE_BF16) return launch_route<uint16_t>(a, stream);
  if (dtype == DSA_DTYPE_F16) return launch_route<_Float16>(a, stream);
  return launch_route<float>(a, stream);
}
