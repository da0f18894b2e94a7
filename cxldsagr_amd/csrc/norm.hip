// The residual stream's sum and its root-mean-square norm, for every row:
//   t = x + r (in 32 bits), y = t w / sqrt(mean t^2 + eps),
// y rounded to 32 bits and then to the element type, as a cast from 64 bits does, t from its 32;
// and, where wanted, the e4m3 codes of the rounded y with a power-of-two scale for every 128
// values, as its exponent (e8m0).
//
// The sum of squares is in 64 bits, y in 46 or more before it is rounded, so that y and its codes
// are those of that cast (a y formed in 32 bits lies on the other side of a rounding border in one
// of some 30,000 values, and of a scale's border now and then, which doubles a whole block's
// step). The 46 bits end at 2^-149: values below 2^-102 of a row's root mean square have fewer.
//
// Bound by memory: a row is read once, kept in registers over the sum, and written once.
#include "quantize_core.h"
#include "../../include/dsa_gfx950.h"

namespace dsa {
namespace {

constexpr int kMaxDim = 16384;
constexpr int kThreads = 512;            // of a work-group at most

struct NormArgs {
  const void* x;
  const void* residual;  // or null
  const void* weight;
  void* values;          // or null
  void* residual_out;    // or null
  uint8_t* codes;        // or null, with scales
  uint8_t* scales;
  int64_t x_stride, residual_stride, tokens;
  int32_t dim, wide_weight;  // wide: fp32, else the rows' type
  double eps, per_dim;       // per_dim: 1 / dim
};

struct Bf16Bits {
  uint16_t v;
};
__device__ __forceinline__ float value_of(Bf16Bits v) { return bf16_to_f32(v.v); }
__device__ __forceinline__ float value_of(_Float16 v) { return (float)v; }
__device__ __forceinline__ float value_of(float v) { return v; }
template <typename T>
__device__ __forceinline__ T rounded(float v) { return (T)v; }
template <>
__device__ __forceinline__ Bf16Bits rounded<Bf16Bits>(float v) { return Bf16Bits{(uint16_t)f32_to_bf16(v)}; }

template <typename T, int kWide>
struct __align__(sizeof(T) * kWide > 16 ? 16 : sizeof(T) * kWide) Pack {
  T v[kWide];
};

// Eight elements that this call does not touch again, and that nothing soon reads, go past the
// caches: rows in, the sum out. What is left of them holds the values and codes, which the next
// operator reads (8,192 rows of 7,168 with codes, 529 MB, 102 us at a copy's rate: on the same
// inputs and outputs 111 -> 104 - 108 us; on inputs that change while the outputs stay the same
// memory, so that the last cache holds part of them, 111 -> 91; the values past the caches too 93,
// the codes too 97; with a read of values and sum behind the call 208 -> 169, 180, 184; 4,096 of
// 4,096 29.7 -> 26.7; short calls as before. Rows of fp32: 187 us, 1.0 GB, 5.3 TB/s).
typedef uint32_t Quad __attribute__((ext_vector_type(4)));
template <typename T>
__device__ __forceinline__ Pack<T, 8> load_once(const Pack<T, 8>* from) {
  using Item = Pack<T, 8>;
  struct {
    Quad part[sizeof(T) / 2];
  } all;
#pragma unroll
  for (int i = 0; i < (int)sizeof(T) / 2; ++i) all.part[i] = __builtin_nontemporal_load(reinterpret_cast<const Quad*>(from) + i);
  return __builtin_bit_cast(Item, all);
}
template <typename T>
__device__ __forceinline__ void store_past(Pack<T, 8>* to, const Pack<T, 8>& v) {
  struct All {
    Quad part[sizeof(T) / 2];
  };
  const All all = __builtin_bit_cast(All, v);
#pragma unroll
  for (int i = 0; i < (int)sizeof(T) / 2; ++i) __builtin_nontemporal_store(all.part[i], reinterpret_cast<Quad*>(to) + i);
}

__device__ __forceinline__ double sum_wave(double v) {
#pragma unroll
  for (int offset = 32; offset > 0; offset >>= 1) v += __shfl_xor(v, offset);
  return v;
}

// The sum over a work-group, by turns of rows in one of two places.
__device__ __forceinline__ double sum_group(double v, double* shared) {
  v = sum_wave(v);
  if ((threadIdx.x & 63) == 0) shared[threadIdx.x >> 6] = v;
  __syncthreads();
  v = shared[0];
  for (int w = 1; w < (int)(blockDim.x >> 6); ++w) v += shared[w];
  return v;
}

// 1 / sqrt(v) in 64 bits: the unit's estimate and a step of the third order. (0 and infinity
// give the estimate's infinity and 0.)
__device__ __forceinline__ double reciprocal_root(double v) {
  const double y = __builtin_amdgcn_rsq(v), r = __builtin_fma(-v * y, y, 1.0);
  const double better = __builtin_fma(y * r, __builtin_fma(0.375, r, 0.5), y);
  return r == r ? better : y;
}

// A product of 64 bits as one of 32. (With contraction the compiler makes its conversion and a
// following one to fp16 a single one, which rounds once.)
__device__ __forceinline__ float rounded_product(double v, double inverse, double weight) {
#pragma clang fp contract(off)
  return (float)(v * inverse * weight);
}

// Items of 8 elements, kItems a thread at most: item i is thread i % threads' item
// i / threads. A work-group goes from row to row with the weight in registers and the next
// row on its way.
template <typename T, int kItems>
__global__ __launch_bounds__(kThreads, kItems * sizeof(T) <= 4 ? 4 : 2) void residual_rms_norm(NormArgs a) {
  using Item = Pack<T, 8>;
  __shared__ double shared[2][kThreads / 64];
  const int threads = blockDim.x, items = a.dim / 8;
  float w[kItems][8];
#pragma unroll
  for (int j = 0; j < kItems; ++j) {
    const int i = threadIdx.x + j * threads;
    if (i >= items) continue;
    if (a.wide_weight) {
      const auto p = reinterpret_cast<const Pack<float, 8>*>(a.weight)[i];
#pragma unroll
      for (int e = 0; e < 8; ++e) w[j][e] = p.v[e];
    } else {
      const Item p = reinterpret_cast<const Item*>(a.weight)[i];
#pragma unroll
      for (int e = 0; e < 8; ++e) w[j][e] = value_of(p.v[e]);
    }
  }
  Item in[kItems], add[kItems];
  auto load = [&](int64_t row) {
    const Item* x = reinterpret_cast<const Item*>(static_cast<const T*>(a.x) + row * a.x_stride);
    const Item* r = reinterpret_cast<const Item*>(static_cast<const T*>(a.residual) + row * a.residual_stride);
#pragma unroll
    for (int j = 0; j < kItems; ++j) {
      const int i = threadIdx.x + j * threads;
      if (i < items) in[j] = load_once(x + i);
      if (i < items && a.residual) add[j] = load_once(r + i);
    }
  };
  load(blockIdx.x);
  int turn = 0;
  for (int64_t row = blockIdx.x; row < a.tokens; row += gridDim.x, turn ^= 1) {
    float t[kItems][8];
    double sum = 0.0;
#pragma unroll
    for (int j = 0; j < kItems; ++j) {
      const int i = threadIdx.x + j * threads;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        t[j][e] = i < items ? value_of(in[j].v[e]) : 0.0f;
        if (i < items && a.residual) t[j][e] += value_of(add[j].v[e]);
        sum = __builtin_fma((double)t[j][e], (double)t[j][e], sum);
      }
    }
    if (row + gridDim.x < a.tokens) load(row + gridDim.x);
    const double mean = __builtin_fma(sum_group(sum, shared[turn]), a.per_dim, a.eps);
    const double inverse = reciprocal_root(mean);
    // t inverse w to 46 bits in pairs of 32 (a third of the time of 64-bit products); where
    // the inverse does not fit a pair, in 64.
    const bool pairs = mean > 0x1p-100 && mean < 0x1p100;
    const float high = (float)inverse, low = (float)(inverse - high);
    auto normed = [&](float v, float weight) {
// (A product that becomes part of the sum would count its rounding twice.)
#pragma clang fp contract(off)
      if (!pairs) return rounded_product(v, inverse, weight);
      const float u = v * high, u_low = __builtin_fmaf(v, low, __builtin_fmaf(v, high, -u));
      const float y = u * weight, both = y + __builtin_fmaf(u_low, weight, __builtin_fmaf(u, weight, -y));
      return both == both ? both : y;  // (an infinity less itself)
    };
    const int64_t base = row * a.dim;
#pragma unroll
    for (int j = 0; j < kItems; ++j) {
      const int i = threadIdx.x + j * threads;
      if (i >= items) continue;
      Item out;
      if (a.residual_out) {
#pragma unroll
        for (int e = 0; e < 8; ++e) out.v[e] = rounded<T>(t[j][e]);
        store_past(reinterpret_cast<Item*>(static_cast<T*>(a.residual_out) + base) + i, out);
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) out.v[e] = rounded<T>(normed(t[j][e], w[j][e]));
      if (a.values) reinterpret_cast<Item*>(static_cast<T*>(a.values) + base)[i] = out;
      if (a.codes) {
        // 16 lanes hold a block of 128 values (the dims are whole blocks).
        float v[8];
        uint32_t top = 0;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          v[e] = value_of(out.v[e]);
          const uint32_t bits = __float_as_uint(v[e]) & 0x7FFFFFFFu;
          top = top > bits ? top : bits;
        }
        const float scale = scale_from_amax_bits(max_abs_bits_reduce<16>(top), true);
        uint32_t lo, hi;
        quantize_eight(v, scale, true, lo, hi);
        *reinterpret_cast<uint2*>(a.codes + base + 8 * i) = make_uint2(lo, hi);
        if ((i & 15) == 0) a.scales[row * (a.dim >> 7) + (i >> 4)] = (uint8_t)(__float_as_uint(scale) >> 23);
      }
    }
  }
}

// Rows whose dims, strides or addresses do not allow vectors: an element at a time, read
// again for the outputs (8,192 rows of 7,167 dims 464 us, where 7,168 take 104).
template <typename T>
__global__ __launch_bounds__(kThreads) void residual_rms_norm_scalar(NormArgs a) {
  __shared__ double shared[2][kThreads / 64];
  int turn = 0;
  for (int64_t row = blockIdx.x; row < a.tokens; row += gridDim.x, turn ^= 1) {
    const T* x = static_cast<const T*>(a.x) + row * a.x_stride;
    const T* r = a.residual ? static_cast<const T*>(a.residual) + row * a.residual_stride : nullptr;
    auto total = [&](int i) { return r ? value_of(x[i]) + value_of(r[i]) : value_of(x[i]); };
    double sum = 0.0;
    for (int i = threadIdx.x; i < a.dim; i += blockDim.x) {
      const double t = total(i);
      sum = __builtin_fma(t, t, sum);
    }
    const double inverse = reciprocal_root(__builtin_fma(sum_group(sum, shared[turn]), a.per_dim, a.eps));
    const int64_t base = row * a.dim;
    for (int i = threadIdx.x; i < a.dim; i += blockDim.x) {
      const float t = total(i);
      if (a.residual_out) static_cast<T*>(a.residual_out)[base + i] = rounded<T>(t);
      const float w = a.wide_weight ? static_cast<const float*>(a.weight)[i] : value_of(static_cast<const T*>(a.weight)[i]);
      if (a.values) static_cast<T*>(a.values)[base + i] = rounded<T>(rounded_product(t, inverse, w));
    }
  }
}

template <typename T>
int launch_norm(const NormArgs& a, bool vector, hipStream_t stream) {
  const int items = vector ? a.dim / 8 : a.dim;
  auto go = [&](auto kernel, int per) {
    int threads = ((items + per - 1) / per + 63) / 64 * 64;
    if (threads > kThreads) threads = kThreads;
    // As many work-groups as the CUs hold at once, 16 waves a CU; each goes on to further rows.
    const int64_t most = (int64_t)device_cu_count() * (16 * 64 / threads);
    hipLaunchKernelGGL(kernel, dim3((unsigned)(a.tokens < most ? a.tokens : most)), dim3(threads), 0, stream, a);
  };
  if (!vector) go(residual_rms_norm_scalar<T>, 1);
  else if (items <= kThreads) go(residual_rms_norm<T, 1>, 1);
  else if (items <= 2 * kThreads) go(residual_rms_norm<T, 2>, 2);
  else go(residual_rms_norm<T, 4>, 4);
  DSA_CHECK_LAUNCH("residual RMS norm");
  return kOk;
}

}  // namespace
}  // namespace dsa

extern "C" int dsa_residual_rms_norm(const void* x, int64_t x_stride, const void* residual, int64_t residual_stride,
                                     int dtype, const void* weight, int weight_dtype, int64_t tokens, int64_t dim,
                                     double eps, void* values, void* residual_out, void* codes, void* scales,
                                     hipStream_t stream) {
  using namespace dsa;
  DSA_CHECK_ARG(dtype >= 0 && dtype <= 2, "unknown element type");
  DSA_CHECK_ARG(weight_dtype == dtype || weight_dtype == DSA_DTYPE_F32, "the weight is fp32 or of the rows' type");
  DSA_CHECK_ARG(tokens >= 0 && dim >= 1 && dim <= kMaxDim, "invalid norm shape (dims from 1 to %d)", kMaxDim);
  DSA_CHECK_ARG(__builtin_isfinite(eps) && eps >= 0, "eps must be finite and nonnegative");
  DSA_CHECK_ARG((codes == nullptr) == (scales == nullptr), "codes and scales come together");
  DSA_CHECK_ARG(residual_out == nullptr || residual != nullptr, "residual_out without a residual");
  if (tokens == 0) return kOk;
  DSA_CHECK_ARG(x && weight, "null pointer");
  NormArgs a{};
  a.x = x, a.residual = residual, a.weight = weight;
  a.values = values, a.residual_out = residual_out;
  a.codes = static_cast<uint8_t*>(codes), a.scales = static_cast<uint8_t*>(scales);
  a.x_stride = x_stride, a.residual_stride = residual_stride, a.tokens = tokens;
  a.dim = (int32_t)dim, a.wide_weight = weight_dtype == DSA_DTYPE_F32;
  a.eps = eps, a.per_dim = 1.0 / (double)dim;
  const int64_t align = dtype == DSA_DTYPE_F32 ? 4 : 8;
  bool vector = dim % 8 == 0 && x_stride % align == 0 && (!residual || residual_stride % align == 0);
  for (const void* p : {x, residual, weight, (const void*)values, (const void*)residual_out})
    vector = vector && reinterpret_cast<uintptr_t>(p) % 16 == 0;
  if (codes)
    DSA_CHECK_ARG(dim % 128 == 0 && vector && reinterpret_cast<uintptr_t>(codes) % 8 == 0,
                  "codes need dims in whole blocks of 128 and rows aligned to 16 bytes");
  if (dtype == DSA_DTYPE_BF16) return launch_norm<Bf16Bits>(a, vector, stream);
  if (dtype == DSA_DTYPE_F16) return launch_norm<_Float16>(a, vector, stream);
  return launch_norm<float>(a, vector, stream);
}
