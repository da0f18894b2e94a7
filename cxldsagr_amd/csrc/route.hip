// Each token's experts from its logits:
//   s = sigmoid(l) or softmax(l), rounded to 32 bits;  b = s + bias (32 bits);
//   of each group of experts the best b, with a bias the sum of its two best (32 bits);
//   the k largest b of the top_groups best groups, in that order, ties to the lower index;
//   w = s, or s / (their sum + 1e-20), times scale.
// Scores are formed in 64 bits and rounded once, so that the order is that of the definition
// and not of some exponential's last bits. A NaN is larger than every number (as in a sort),
// so that it shows in the weights.
//
// kLanes lanes take a token, some lanes a group: a group's experts are cut into runs of
// `per`, one for each of `parts` lanes (a power of two), so that every count of experts and
// groups fits. An expert's rank is one number of 42 bits, its b as an ordered integer above
// its index counted down, held as a positive double of those bits: v_max_f64 compares them
// in one instruction, and no two are equal. k times the largest is found over the lanes and
// struck out.
#include "dsa_common.h"
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
  int32_t k, groups, top_groups, size, parts, per, softmax, renormalize;
  float scale;
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

// op over the lanes of a token, in all of them.
template <int kLanes, typename Op>
__device__ __forceinline__ double over_lanes(double v, Op op) {
  auto step = [&](auto move) {
    const uint64_t b = __builtin_bit_cast(uint64_t, v);
    const uint32_t lo = move((uint32_t)b), hi = move((uint32_t)(b >> 32));
    v = op(v, __builtin_bit_cast(double, (uint64_t)hi << 32 | lo));
  };
  step([](uint32_t w) { return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)w, 0xB1, 0xF, 0xF, false); });
  step([](uint32_t w) { return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)w, 0x4E, 0xF, 0xF, false); });
  step([](uint32_t w) { return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)w, 0x141, 0xF, 0xF, false); });
  step([](uint32_t w) { return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)w, 0x140, 0xF, 0xF, false); });
  if constexpr (kLanes == 64) {
    step([](uint32_t w) { return (uint32_t)__shfl_xor((int)w, 16); });
    step([](uint32_t w) { return (uint32_t)__shfl_xor((int)w, 32); });
  }
  return v;
}

template <typename T, int kLanes, int kSlots>
__global__ __launch_bounds__(kThreads) void route(RouteArgs a) {
  constexpr int kTokens = kThreads / kLanes;
  __shared__ float chosen_score[kTokens][kMaxChoices];
  __shared__ int32_t chosen_id[kTokens][kMaxChoices];
  const int l = threadIdx.x % kLanes, local = threadIdx.x / kLanes;
  const int64_t own = (int64_t)blockIdx.x * kTokens + local;
  const bool live = own < a.tokens;
  const T* logits = static_cast<const T*>(a.logits) + (live ? own : a.tokens - 1) * a.stride;
  const int group = l / a.parts, from = l % a.parts * a.per;
  const int end = group < a.groups ? (a.size - from < a.per ? a.size - from : a.per) : 0;  // this lane's slots
  const int first = group * a.size + from;

  float s[kSlots];
#pragma unroll
  for (int i = 0; i < kSlots; ++i) s[i] = i < end ? value_of(logits[first + i]) : -__builtin_inff();
  if (a.softmax) {
    float top = s[0];
#pragma unroll
    for (int i = 1; i < kSlots; ++i) top = fmaxf(top, s[i]);
    const double most = over_lanes<kLanes>((double)top, [](double x, double y) { return fmax(x, y); });
    double e[kSlots], sum = 0.0;
#pragma unroll
    for (int i = 0; i < kSlots; ++i) {
      e[i] = i < end ? exp((double)s[i] - most) : 0.0;
      sum += e[i];
    }
    sum = over_lanes<kLanes>(sum, [](double x, double y) { return x + y; });
#pragma unroll
    for (int i = 0; i < kSlots; ++i) s[i] = (float)(e[i] / sum);
  } else {
#pragma unroll
    for (int i = 0; i < kSlots; ++i)
      if (i < end) s[i] = (float)(1.0 / (1.0 + exp(-(double)s[i])));
  }

  uint32_t key[kSlots];
#pragma unroll
  for (int i = 0; i < kSlots; ++i) key[i] = i < end ? ordered(a.bias ? s[i] + a.bias[first + i] : s[i]) : 0u;
  if (a.top_groups < a.groups) {
    uint32_t one = 0, two = 0;  // the group's best and next
#pragma unroll
    for (int i = 0; i < kSlots; ++i) {
      const uint32_t less = key[i] < one ? key[i] : one;
      one = key[i] < one ? one : key[i];
      two = two > less ? two : less;
    }
    for (int offset = 1; offset < a.parts; offset <<= 1) {
      const uint32_t o1 = (uint32_t)__shfl_xor((int)one, offset), o2 = (uint32_t)__shfl_xor((int)two, offset);
      const uint32_t less = one < o1 ? one : o1, second = two > o2 ? two : o2;
      one = one > o1 ? one : o1;
      two = less > second ? less : second;
    }
    const uint32_t mine = a.bias && two ? ordered(from_ordered(one) + from_ordered(two)) : one;
    int better = 0;
    for (int g = 0; g < a.groups; ++g) {
      const uint32_t other = (uint32_t)__shfl((int)mine, g * a.parts, kLanes);
      better += other > mine || (other == mine && g < group);
    }
    if (better >= a.top_groups) {
#pragma unroll
      for (int i = 0; i < kSlots; ++i) key[i] = 0u;
    }
  }

  double rank[kSlots];
#pragma unroll
  for (int i = 0; i < kSlots; ++i)
    rank[i] = __builtin_bit_cast(double, key[i] ? (uint64_t)key[i] << 30 | (uint64_t)(1023 - (first + i)) << 20 : 0ull);
  for (int c = 0; c < a.k; ++c) {
    double best = rank[0];
#pragma unroll
    for (int i = 1; i < kSlots; ++i) best = fmax(best, rank[i]);
    best = over_lanes<kLanes>(best, [](double x, double y) { return fmax(x, y); });
#pragma unroll
    for (int i = 0; i < kSlots; ++i)
      if (rank[i] == best) {
        chosen_score[local][c] = s[i];
        chosen_id[local][c] = first + i;
        rank[i] = 0.0;
      }
  }
  __syncthreads();
  if (!live) return;
  float factor = a.scale;
  float sum = 0.0f;
  for (int c = 0; c < a.k; ++c) sum += chosen_score[local][c];
  for (int c = l; c < a.k; c += kLanes) {
    const float w = chosen_score[local][c];
    a.weights[own * a.k + c] = (a.renormalize ? w / (sum + 1e-20f) : w) * factor;
    a.ids[own * a.k + c] = chosen_id[local][c];
  }
}

template <typename T>
int launch_route(RouteArgs a, hipStream_t stream) {
  // Lanes of a token, of a group, and a lane's experts.
  auto plan = [&](int lanes) {
    a.parts = 1;
    while (2 * a.parts * a.groups <= lanes) a.parts *= 2;
    a.per = (a.size + a.parts - 1) / a.parts;
  };
  auto go = [&](auto kernel, int lanes) {
    const int64_t tokens = kThreads / lanes;
    hipLaunchKernelGGL(kernel, dim3((unsigned)((a.tokens + tokens - 1) / tokens)), dim3(kThreads), 0, stream, a);
  };
  plan(64);
  if (a.per <= 4) go(route<T, 64, 4>, 64);
  else if (a.per <= 16) go(route<T, 64, 16>, 64);
  else go(route<T, 64, 32>, 64);
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
  DSA_CHECK_ARG(grid_fits(tokens, 64), "too many tokens for one launch");
  if (tokens == 0) return kOk;
  DSA_CHECK_ARG(logits && weights && ids, "null pointer");
  RouteArgs a{};
  a.logits = logits, a.bias = bias, a.weights = weights, a.ids = ids;
  a.stride = stride, a.tokens = tokens, a.k = (int32_t)k;
  a.groups = (int32_t)groups, a.top_groups = (int32_t)top_groups, a.size = (int32_t)(experts / groups);
  a.softmax = softmax != 0, a.renormalize = renormalize != 0, a.scale = (float)scale;
  if (dtype == DSA_DTYPE_BF16) return launch_route<uint16_t>(a, stream);
  if (dtype == DSA_DTYPE_F16) return launch_route<_Float16>(a, stream);
  return launch_route<float>(a, stream);
}
