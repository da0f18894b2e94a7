// The routed experts' gated MLP in 8 bits. For token t and each of its choices j, expert e:
//   g = x Wg_e, u = x Wu_e,  h = g / (1 + exp(-g)) * u  (32 bits),  q = e4m3 codes of h,
//   y_j = q Wd_e,            out_t = sum_j w_j y_j,
// x, q and the weights in e4m3 with a power-of-two scale (e8m0) for every 128 values of a
// row, and every 128 by 128 of a weight.
//
// Four launches:
//  1. group: the (token, choice) pairs of each expert, in token order, and row tiles of them;
//  2. up: row tiles times gate and up, h, its codes and scales;
//  3. down: row tiles times down, y in 16 bits with a power of two for every 64 values of a
//     row (its largest value just below 2^15 as fp16: 11 bits of each value; as bf16, 8, the
//     result would be sqrt 2 times as far from the formula as its own rounding puts it);
//  4. join: each token's y, weighted, in 32 bits, in the order of its choices.
// No atomics on values: results do not depend on the order of work-groups.
//
// The products run on v_mfma_scale_f32_16x16x128_f8f6f4, weights as the first operand (rows:
// 16 of a weight's), tokens as the second (columns), so that a lane's four results are
// neighbours in the output's row. The instruction multiplies by each operand's scale, a
// power of two per 32 values along K: the blocks of 128 cost nothing beyond that. Sums are
// in 32 bits. Weights are laid out as the instruction reads them (ExpertWeights): a tile of
// 16 rows by 128 is 2 KB, two planes of 16 bytes a lane, read by one wave straight into
// registers; tiles of gate and up alternate, so that a lane holds g and u of the same h.
#include "attention_core.h"
#include "quantize_core.h"
#include "../../include/dsa_gfx950.h"

namespace dsa {
namespace {

typedef int v8i __attribute__((ext_vector_type(8)));

constexpr int kBlock = 128;                 // values that share a scale; K of a step
constexpr int kTile = 16 * kBlock;          // bytes of a weight's tile
constexpr int kWaveCols = 64;               // weight rows (output columns) of a wave: four tiles
constexpr int kMaxExperts = 1024;
constexpr int kGroupThreads = 1024;

// 32 codes of a lane from its 16 bytes of both planes.
__device__ __forceinline__ v8i joined(v4u low, v4u high) {
  return __builtin_bit_cast(v8i, __builtin_shufflevector(low, high, 0, 1, 2, 3, 4, 5, 6, 7));
}

// The scales are bytes kW and kX of their words.
template <int kW = 0, int kX = 0>
__device__ __forceinline__ v4f product(v8i w, v8i x, v4f c, uint32_t w_scale, uint32_t x_scale) {
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(w, x, c, 0, 0, kW, (int)w_scale, kX, (int)x_scale);
}

// ------------------------------------------------------------ 1. groups --
struct Tile {
  int32_t expert, row, rows;
  int32_t first, count;  // the expert's tiles
  int32_t unused[3];
};

struct GroupArgs {
  const int32_t* ids;   // [pairs]
  int32_t* order;       // [pairs]: the pair of a row
  int32_t* place;       // [pairs]: the row of a pair (of this call's experts)
  Tile* tiles;
  int32_t* tile_count;
  int32_t pairs, first, experts, tile_rows;
};

// Work-group e lists expert e's pairs. Each counts all experts' (in LDS), so that none waits
// for another: rows and tiles of the experts before e are sums over the counts. A wave takes
// a run of the pairs, so that a pair's row is the sum of what was found before it.
__global__ __launch_bounds__(kGroupThreads) void group_pairs(GroupArgs a) {
  __shared__ uint32_t counts[kMaxExperts];
  __shared__ uint32_t of_wave[kGroupThreads / 64][3];
  const int expert = blockIdx.x, wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  constexpr int kWaves = kGroupThreads / 64;
  for (int i = threadIdx.x; i < a.experts; i += kGroupThreads) counts[i] = 0;
  __syncthreads();
  const int run = ((a.pairs + kWaves - 1) / kWaves + 63) / 64 * 64;
  const int64_t begin = (int64_t)wave * run, end = begin + run < a.pairs ? begin + run : a.pairs;
  uint32_t found = 0;
  for (int64_t i = begin + lane; i < end; i += 64) {
    const uint32_t e = (uint32_t)a.ids[i] - (uint32_t)a.first;
    if (e < (uint32_t)a.experts) atomicAdd(&counts[e], 1u);
    found += e == (uint32_t)expert;
  }
  found = sum_lanes(found);
  __syncthreads();
  // Rows and tiles before this expert's, this thread's expert being i.
  const int i = threadIdx.x;
  const uint32_t n = i < a.experts ? counts[i] : 0u;
  const uint32_t tiles_of = (n + a.tile_rows - 1) / a.tile_rows;
  const uint32_t rows = sum_lanes(i < expert ? n : 0u), tiles = sum_lanes(i < expert ? tiles_of : 0u);
  if (lane == 0) of_wave[wave][0] = rows, of_wave[wave][1] = tiles, of_wave[wave][2] = found;
  __syncthreads();
  uint32_t row = 0, tile = 0, before = 0;
  for (int w = 0; w < kWaves; ++w) {
    row += of_wave[w][0], tile += of_wave[w][1];
    if (w < wave) before += of_wave[w][2];
  }
  const uint32_t own = counts[expert], own_tiles = (own + a.tile_rows - 1) / a.tile_rows;
  for (uint32_t t = threadIdx.x; t < own_tiles; t += kGroupThreads) {
    const uint32_t at = t * a.tile_rows, left = own - at;
    a.tiles[tile + t] = Tile{expert, (int32_t)(row + at), (int32_t)(left < (uint32_t)a.tile_rows ? left : a.tile_rows),
                             (int32_t)tile, (int32_t)own_tiles, {}};
  }
  if (expert == a.experts - 1 && threadIdx.x == 0) *a.tile_count = (int32_t)(tile + own_tiles);
  uint32_t next = row + before;
  for (int64_t base = begin; base < end; base += 64) {
    const int64_t p = base + lane;
    const bool mine = p < end && (uint32_t)a.ids[p] - (uint32_t)a.first == (uint32_t)expert;
    const uint64_t all = __ballot(mine);
    if (mine) {
      const uint32_t to = next + (uint32_t)__popcll(all & ((1ull << lane) - 1));
      a.order[to] = (int32_t)p;
      a.place[p] = (int32_t)to;
    }
    next += (uint32_t)__popcll(all);
  }
}

// ------------------------------------------------------ 2, 3. products --
struct ProductArgs {
  const uint8_t* x;        // rows of `depth` codes: tokens (up), pairs in order (down)
  const uint8_t* x_scale;  // [rows, depth / 128]
  const int32_t* order;
  const uint8_t* w;        // [experts][columns / 16][depth / 128][2048]
  const uint8_t* w_scale;  // [experts][columns / 128][depth / 128]
  const Tile* tiles;
  const int32_t* tile_count;
  uint8_t* codes;          // up: h [pairs, inner] and its scales
  uint8_t* scales;
  uint16_t* y;             // down: [pairs, columns] fp16, and its powers [pairs, columns / 64]
  uint8_t* powers;
  int32_t depth, columns, choices, column_blocks;
};

__device__ __forceinline__ float silu(float g) {
  return g * __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(g * -kLog2E));
}

__device__ __forceinline__ uint32_t max_over_groups(uint32_t v) {
  const auto a = __builtin_amdgcn_permlane16_swap(v, v, false, false);
  v = a[0] > a[1] ? a[0] : a[1];
  const auto b = __builtin_amdgcn_permlane32_swap(v, v, false, false);
  return b[0] > b[1] ? b[0] : b[1];
}

// h of a work-group's rows and 128 columns (a wave's 32 of them in acc: tiles of gate and
// up in turn), its codes and scales. amax: [4][16 kRows] words of LDS that no wave uses.
template <int kRows>
__device__ __forceinline__ void store_hidden(const ProductArgs& a, const Tile& tile, const v4f (&acc)[kRows][4], int block,
                                             uint32_t* amax) {
  const int wave = threadIdx.x >> 6, r = threadIdx.x & 15, g = (threadIdx.x & 63) >> 4;
  const int64_t inner = a.columns / 2;
  float h[kRows][8];
#pragma unroll
  for (int m = 0; m < kRows; ++m) {
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      h[m][i] = silu(acc[m][i >> 2 << 1][i & 3]) * acc[m][(i >> 2 << 1) + 1][i & 3];
      const uint32_t bits = __float_as_uint(h[m][i]) & 0x7FFFFFFFu;
      top = top > bits ? top : bits;
    }
    top = max_over_groups(top);
    if (g == 0) amax[(wave * kRows + m) * 16 + r] = top;
  }
  __syncthreads();
#pragma unroll
  for (int m = 0; m < kRows; ++m) {
    uint32_t top = 0;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const uint32_t of = amax[(w * kRows + m) * 16 + r];
      top = top > of ? top : of;
    }
    const float scale = scale_from_amax_bits(top, true);
    if (16 * m + r >= tile.rows) continue;
    const int64_t row = tile.row + 16 * m + r;
    uint32_t lo, hi;
    quantize_eight(h[m], scale, true, lo, hi);
    uint8_t* to = a.codes + row * inner + block * 128 + wave * 32 + 4 * g;
    *reinterpret_cast<uint32_t*>(to) = lo;
    *reinterpret_cast<uint32_t*>(to + 16) = hi;
    if (wave == 0 && g == 0) a.scales[row * (inner / kBlock) + block] = (uint8_t)(__float_as_uint(scale) >> 23);
  }
}

// y of a wave's rows and 64 columns from `column` on.
template <int kRows>
__device__ __forceinline__ void store_result(const ProductArgs& a, const Tile& tile, const v4f (&acc)[kRows][4], int column) {
  const int r = threadIdx.x & 15, g = (threadIdx.x & 63) >> 4;
#pragma unroll
  for (int m = 0; m < kRows; ++m) {
    // The largest finite magnitude of the row's 64 values, its power of two.
    uint32_t top = 0;
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t bits = __float_as_uint(acc[m][t][i]) & 0x7FFFFFFFu;
        top = bits < 0x7F800000u && bits > top ? bits : top;
      }
    top = max_over_groups(top);
    // (At least 2^-112: a smaller row of 64 keeps steps of 2^-136.)
    const uint32_t power = (top >> 23) < 15u ? 15u : top >> 23;
    const float factor = __uint_as_float((268u - power) << 23);
    if (column >= a.columns || 16 * m + r >= tile.rows) continue;
    const int64_t row = tile.row + 16 * m + r;
    uint16_t* to = a.y + row * a.columns + column + 4 * g;
#pragma unroll
    for (int t = 0; t < 4; ++t)
      *reinterpret_cast<uint2*>(to + 16 * t) =
          make_uint2(F16::pack(acc[m][t][0] * factor, acc[m][t][1] * factor),
                     F16::pack(acc[m][t][2] * factor, acc[m][t][3] * factor));
    if (g == 0) a.powers[row * (a.columns / kWaveCols) + column / kWaveCols] = (uint8_t)power;
  }
}

// The parts of the weight that a wave of `column` (past the end: of the last) reads.
struct WaveWeight {
  const uint8_t* codes;          // this lane's 16 bytes of the first tile
  const uint8_t* scale[2];       // of even and odd tiles (up: gate's and up's), a byte a step
};
template <bool kUp>
__device__ __forceinline__ WaveWeight weight_of(const ProductArgs& a, int expert, int block, int column, int steps) {
  const int at = column < a.columns ? column : a.columns - kWaveCols;
  WaveWeight w;
  w.codes = a.w + ((int64_t)expert * (a.columns / 16) + at / 16) * steps * kTile + (threadIdx.x & 63) * 16;
  const uint8_t* scale = a.w_scale + (int64_t)expert * (a.columns / kBlock) * steps;
  w.scale[0] = scale + (int64_t)(kUp ? block : at / kBlock) * steps;
  w.scale[1] = kUp ? w.scale[0] + (int64_t)(a.columns / 256) * steps : w.scale[0];
  return w;
}

// The weight's 64 rows of one step.
__device__ __forceinline__ void load_weight(v8i (&to)[4], const uint8_t* codes, int steps, int s) {
#pragma unroll
  for (int t = 0; t < 4; ++t) {
    const v4u* from = reinterpret_cast<const v4u*>(codes + ((int64_t)t * steps + s) * kTile);
    to[t] = joined(from[0], from[64]);
  }
}

// Few rows: kRows 16-row tiles by 4 waves of 64 columns, every wave streaming its own part
// of the weight, and the tokens' codes, through registers. What bounds it is reading the
// weight.
template <int kRows, bool kUp>
__global__ __launch_bounds__(256) void expert_product(ProductArgs a) {
  const int tile_at = blockIdx.x / a.column_blocks, block = blockIdx.x % a.column_blocks;
  if (tile_at >= *a.tile_count) return;
  const Tile tile = a.tiles[tile_at];
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4;
  const int column = block * 256 + wave * kWaveCols;  // of the packed weight
  const int steps = a.depth / kBlock;
  __shared__ uint32_t amax[kUp ? 4 * 16 * kRows : 1];

  const uint8_t* x[kRows];
  const uint8_t* xs[kRows];
#pragma unroll
  for (int m = 0; m < kRows; ++m) {
    const int in = 16 * m + r;
    int64_t row = tile.row + (in < tile.rows ? in : tile.rows - 1);
    if constexpr (kUp) row = a.order[row] / a.choices;
    x[m] = a.x + row * a.depth + g * 16;
    xs[m] = a.x_scale + row * steps;
  }
  const WaveWeight w = weight_of<kUp>(a, tile.expert, block, column, steps);

  v4f acc[kRows][4] = {};
  for (int s = 0; s < steps; ++s) {
    v8i wv[4];
    load_weight(wv, w.codes, steps, s);
    const int s0 = w.scale[0][s], s1 = w.scale[1][s];
#pragma unroll
    for (int m = 0; m < kRows; ++m) {
      const v4u* from = reinterpret_cast<const v4u*>(x[m] + s * kBlock);
      const v8i xv = joined(from[0], from[4]);
      const int sx = xs[m][s];
#pragma unroll
      for (int t = 0; t < 4; ++t) acc[m][t] = product(wv[t], xv, acc[m][t], t & 1 ? s1 : s0, sx);
    }
  }
  if constexpr (kUp) store_hidden<kRows>(a, tile, acc, block, amax);
  else store_result<kRows>(a, tile, acc, column);
}

// Many rows: 16 kRows rows by 256 columns. Each wave keeps its 64 columns of the weight in
// registers, a step ahead; the rows' codes go into LDS straight from memory (two steps
// ahead, four buffers), where all four waves read them, three 16-row tiles ahead of their
// products. Half-way through a step the waves meet: from there on the next step's rows may
// be read. A row's eight 16-byte parts are turned by its index, so that eight rows' reads of
// one part fall on different banks.
// Per step of 128 a CU's matrix units take 8 kRows 16 clocks, its LDS 10 kRows 8 (four waves'
// reads and one write of 2 kRows KB at 128 bytes), its path to L2 half as many.
constexpr int kMaxWideSteps = 120;
template <int kRows>
struct WideLds {
  alignas(16) uint8_t rows[4][16 * kRows * kBlock];
  alignas(16) uint8_t scales[kMaxWideSteps][16][kRows];  // a row's tile last: one read holds all
  alignas(4) uint8_t weight_scales[kMaxWideSteps][2];
};

template <int kRows, bool kUp>
__global__ __launch_bounds__(256, kRows <= 8 ? 2 : 1) void expert_product_wide(ProductArgs a) {
  __shared__ WideLds<kRows> lds;
  // Work-groups go round the eight XCDs: each takes a run of the work, in which an expert's
  // row tiles are neighbours and read the same columns of its weight through one L2.
  const int64_t all = (int64_t)*a.tile_count * a.column_blocks, each = (all + 7) / 8;
  const int64_t at = (int64_t)(blockIdx.x & 7) * each + (blockIdx.x >> 3);
  if ((blockIdx.x >> 3) >= each || at >= all) return;
  Tile tile = a.tiles[at / a.column_blocks];
  const int64_t within = at - (int64_t)tile.first * a.column_blocks;
  const int block = (int)(within / tile.count);
  tile = a.tiles[tile.first + within % tile.count];

  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4;
  const int column = block * 256 + wave * kWaveCols;
  const int steps = a.depth / kBlock;
  const WaveWeight w = weight_of<kUp>(a, tile.expert, block, column, steps);

  // This lane's parts of the rows that its wave fetches: 4 kRows rows, eight a load.
  constexpr int kLoads = kRows / 2;
  uint64_t from[kLoads];
#pragma unroll
  for (int i = 0; i < kLoads; ++i) {
    const int in = (wave * kLoads + i) * 8 + (lane >> 3);
    int64_t row = tile.row + (in < tile.rows ? in : tile.rows - 1);
    if constexpr (kUp) row = a.order[row] / a.choices;
    from[i] = (uint64_t)(a.x + row * a.depth + (((lane & 7) ^ (in & 7)) << 4));
  }
  const uint32_t lds_rows = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint8_t*)&lds.rows[0][0];
  auto fetch = [&](int buffer) {
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      const uint32_t to = lds_rows + buffer * (16 * kRows * kBlock) + (wave * kLoads + i) * 1024;
      asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off"
                   ::"s"(__builtin_amdgcn_readfirstlane(to)), "v"(from[i]) : "memory", "m0");
    }
  };
  auto advance = [&](bool on) {
#pragma unroll
    for (int i = 0; i < kLoads; ++i) from[i] += on ? kBlock : 0;
  };
  fetch(0);
  advance(steps > 1);
  fetch(1);
  v8i now[4];
  load_weight(now, w.codes, steps, 0);

  // The rows' and the weight's scales of all steps.
  {
    constexpr int kPer = 256 / (16 * kRows);  // threads of a row
    const int in = threadIdx.x / kPer, part = threadIdx.x % kPer;
    int64_t row = tile.row + (in < tile.rows ? in : tile.rows - 1);
    if constexpr (kUp) row = a.order[row] / a.choices;
    const uint8_t* xs = a.x_scale + row * steps;
#pragma unroll 8
    for (int s = part; s < steps; s += kPer) lds.scales[s][in & 15][in >> 4] = xs[s];
    // (Down: of a block of 128 columns each pair of waves, up: of gate and up.)
    const WaveWeight other = weight_of<kUp>(a, tile.expert, block, block * 256 + 128, steps);
    const WaveWeight one = weight_of<kUp>(a, tile.expert, block, block * 256, steps);
    for (int s = threadIdx.x; s < steps; s += 256) {
      lds.weight_scales[s][0] = one.scale[0][s];
      lds.weight_scales[s][1] = (kUp ? one.scale[1] : other.scale[0])[s];
    }
  }
  wait_loads<0>();
  lds_barrier();

  const uint32_t lane_at = lds_rows + r * kBlock + ((g ^ (r & 7)) << 4);
  // Tiles of rows in registers: those ahead of the products hide the LDS (with two waves a
  // SIMD one is enough, and fits).
  constexpr int kRing = kRows <= 8 ? 2 : 4, kAhead = kRing - 1;
  v8i x[kRing];
  auto read = [&](uint32_t buffer, int m) {
    const uint32_t from = buffer * (16 * kRows * kBlock) + m * 16 * kBlock;
    return joined(lds_load<v4u>(lane_at + from), lds_load<v4u>((lane_at ^ 64) + from));
  };
  typedef uint32_t RowScales __attribute__((ext_vector_type(kRows / 4)));
  auto scales_of = [&](int s) { return *reinterpret_cast<const RowScales*>(&lds.scales[s][r][0]); };
  auto weight_scales_of = [&](int s) {
    const uint32_t both = *reinterpret_cast<const uint16_t*>(&lds.weight_scales[s][0]);
    return kUp ? both : both >> (wave >> 1 << 3);
  };
#pragma unroll
  for (int m = 0; m < kAhead; ++m) x[m] = read(0, m);
  RowScales xs = scales_of(0);
  uint32_t ws = weight_scales_of(0);

  v4f acc[kRows][4] = {};
#pragma unroll 1
  for (int s = 0; s < steps; ++s) {
    const int ahead = s + 1 < steps ? s + 1 : s;
    v8i next[4];
    const RowScales xs_next = scales_of(ahead);
    const uint32_t ws_next = weight_scales_of(ahead);
    static_for<kRows>([&](auto index) {
      constexpr int m = decltype(index)::value;
      __builtin_amdgcn_sched_barrier(0);
      if constexpr (m == 1) {
        // Behind the first products, which wait for this step's weight: what is asked for
        // here would be waited for there. (At the end the last rows come again, into buffers
        // that are not read.)
        advance(s + 2 < steps);
        fetch((s + 2) & 3);
        load_weight(next, w.codes, steps, ahead);
        __builtin_amdgcn_sched_barrier(0);
      }
      if constexpr (m == kRows / 2) {
        // This wave's rows of the next step have come, and everyone's.
        wait_loads<kLoads + 8>();
        __builtin_amdgcn_s_barrier();
        __builtin_amdgcn_sched_barrier(0);
      }
      x[(m + kAhead) % kRing] = m + kAhead < kRows ? read(s & 3, m + kAhead) : read((s + 1) & 3, m + kAhead - kRows);
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        if (kUp && (t & 1)) acc[m][t] = product<1, m & 3>(now[t], x[m % kRing], acc[m][t], ws, xs[m / 4]);
        else acc[m][t] = product<0, m & 3>(now[t], x[m % kRing], acc[m][t], ws, xs[m / 4]);
      }
    });
#pragma unroll
    for (int t = 0; t < 4; ++t) now[t] = next[t];
    xs = xs_next;
    ws = ws_next;
  }
  // (What is still on its way into LDS has to land before the LDS is another's.)
  wait_loads<0>();

  if constexpr (kUp) {
    __syncthreads();
    store_hidden<kRows>(a, tile, acc, block, reinterpret_cast<uint32_t*>(&lds.rows[0][0]));
  } else {
    store_result<kRows>(a, tile, acc, column);
  }
}

// --------------------------------------------------------------- 4. join --
struct JoinArgs {
  const int32_t* ids;
  const int32_t* place;
  const float* weights;
  const uint16_t* y;
  const uint8_t* powers;
  void* out;
  int32_t choices, first, experts, dim, groups_per_token;
};

struct Bf16Bits {
  uint16_t v;
};
template <typename T>
__device__ __forceinline__ T rounded(float v) { return (T)v; }
template <>
__device__ __forceinline__ Bf16Bits rounded<Bf16Bits>(float v) { return Bf16Bits{(uint16_t)f32_to_bf16(v)}; }

// Eight columns of a token a thread.
template <typename T>
__global__ __launch_bounds__(256) void join_choices(JoinArgs a) {
  struct __align__(16) Eight {
    T v[8];
  };
  const int64_t token = blockIdx.x / a.groups_per_token;
  const int column = ((int)(blockIdx.x % a.groups_per_token) * 256 + (int)threadIdx.x) * 8;
  if (column >= a.dim) return;
  float sum[8] = {};
  for (int c = 0; c < a.choices; ++c) {
    const int64_t pair = token * a.choices + c;
    if ((uint32_t)a.ids[pair] - (uint32_t)a.first >= (uint32_t)a.experts) continue;
    const int64_t row = a.place[pair];
    const float weight = a.weights[pair];
    const v8hf y = *reinterpret_cast<const v8hf*>(a.y + row * a.dim + column);
    const uint32_t power = a.powers[row * (a.dim / kWaveCols) + column / kWaveCols];
    const float unit = __uint_as_float((power - 14u) << 23);
#pragma unroll
    for (int i = 0; i < 8; ++i) sum[i] += (float)y[i] * unit * weight;
  }
  Eight out;
#pragma unroll
  for (int i = 0; i < 8; ++i) out.v[i] = rounded<T>(sum[i]);
  *reinterpret_cast<Eight*>(static_cast<T*>(a.out) + token * a.dim + column) = out;
}

// ----------------------------------------------------------------- calls --
struct Plan {
  int64_t pairs, tiles;       // of the longest call, and its row tiles at most
  int rows;                   // 16-row parts of a tile
  // Offsets of the workspace's parts.
  int64_t count, list, order, place, codes, scales, y, powers, bytes;
};

Plan plan_of(int64_t tokens, int64_t choices, int64_t dim, int64_t inner, int64_t experts, int64_t total) {
  Plan p{};
  p.pairs = tokens * choices;
  // Rows of an expert, on average; tiles of about twice that.
  const int64_t mean = p.pairs / total;
  p.rows = mean <= 6 ? 1 : mean <= 16 ? 2 : mean <= 40 ? 4 : mean <= 128 ? 8 : 16;
  if (dim > kMaxWideSteps * kBlock || inner > kMaxWideSteps * kBlock) p.rows = p.rows < 4 ? p.rows : 4;
  const int64_t size = 16 * p.rows;
  p.tiles = p.pairs / size + (experts < p.pairs ? experts : p.pairs);
  if (p.tiles > p.pairs) p.tiles = p.pairs;
  int64_t at = 0;
  auto part = [&](int64_t bytes) {
    const int64_t here = at;
    at += (bytes + 255) / 256 * 256;
    return here;
  };
  p.count = part(4);
  p.list = part(p.tiles * (int64_t)sizeof(Tile));
  p.order = part(p.pairs * 4);
  p.place = part(p.pairs * 4);
  p.codes = part(p.pairs * inner);
  p.scales = part(p.pairs * (inner / kBlock));
  p.y = part(p.pairs * dim * 2);
  p.powers = part(p.pairs * (dim / kWaveCols));
  p.bytes = at;
  return p;
}

int check_shape(int64_t tokens, int64_t choices, int64_t dim, int64_t inner, int64_t experts, int64_t total) {
  DSA_CHECK_ARG(dim >= kBlock && dim % kBlock == 0 && dim <= 32768 && inner >= kBlock && inner % kBlock == 0 &&
                    inner <= 32768,
                "dims must be whole blocks of 128, 32768 at most");
  DSA_CHECK_ARG(experts >= 1 && experts <= kMaxExperts && total >= experts, "experts must number 1 to %d", kMaxExperts);
  DSA_CHECK_ARG(choices >= 1 && choices <= 64, "choices must number 1 to 64");
  DSA_CHECK_ARG(tokens >= 0 && tokens <= (1 << 22), "tokens must number 0 to 2^22");
  return kOk;
}

template <bool kUp>
int launch_product(const ProductArgs& a, const Plan& p, hipStream_t stream) {
  auto go = [&](auto kernel, int64_t groups) {
    hipLaunchKernelGGL(kernel, dim3((unsigned)groups), dim3(256), 0, stream, a);
  };
  const int64_t groups = p.tiles * a.column_blocks;
  if (p.rows == 1) go(expert_product<1, kUp>, groups);
  else if (p.rows == 2) go(expert_product<2, kUp>, groups);
  else if (p.rows == 4) go(expert_product<4, kUp>, groups);
  else if (p.rows == 8) go(expert_product_wide<8, kUp>, (groups + 7) / 8 * 8);
  else go(expert_product_wide<16, kUp>, (groups + 7) / 8 * 8);
  DSA_CHECK_LAUNCH("expert product");
  return kOk;
}

}  // namespace
}  // namespace dsa

extern "C" int dsa_expert_mlp_workspace_bytes(int64_t tokens, int64_t choices, int64_t dim, int64_t inner,
                                              int64_t experts, int64_t total, int64_t* bytes) {
  using namespace dsa;
  DSA_CHECK_ARG(bytes, "null pointer");
  if (const int status = check_shape(tokens, choices, dim, inner, experts, total)) return status;
  *bytes = plan_of(tokens, choices, dim, inner, experts, total).bytes;
  return kOk;
}

extern "C" int dsa_expert_mlp_fp8(const void* x, const void* x_scale, int64_t tokens, int64_t dim, int64_t inner,
                                  const void* gate_up, const void* gate_up_scale, const void* down,
                                  const void* down_scale, int64_t experts, int64_t first, int64_t total,
                                  const int32_t* ids, const float* weights, int64_t choices, void* out, int dtype,
                                  void* workspace, int64_t workspace_bytes, hipStream_t stream) {
  using namespace dsa;
  if (const int status = check_shape(tokens, choices, dim, inner, experts, total)) return status;
  DSA_CHECK_ARG(dtype >= 0 && dtype <= 2, "unknown element type");
  DSA_CHECK_ARG(first >= 0 && first <= (1 << 30), "first must be 0 to 2^30");
  if (tokens == 0) return kOk;
  DSA_CHECK_ARG(x && x_scale && gate_up && gate_up_scale && down && down_scale && ids && weights && out && workspace,
                "null pointer");
  for (const void* p : {x, gate_up, down, (const void*)out, (const void*)workspace})
    DSA_CHECK_ARG(reinterpret_cast<uintptr_t>(p) % 16 == 0, "codes, weights, out and workspace must be 16-byte aligned");
  const Plan p = plan_of(tokens, choices, dim, inner, experts, total);
  DSA_CHECK_ARG(workspace_bytes >= p.bytes, "workspace of %lld bytes is smaller than the %lld needed",
                (long long)workspace_bytes, (long long)p.bytes);
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  Tile* tiles = reinterpret_cast<Tile*>(ws + p.list);
  int32_t* count = reinterpret_cast<int32_t*>(ws + p.count);
  int32_t* order = reinterpret_cast<int32_t*>(ws + p.order);
  int32_t* place = reinterpret_cast<int32_t*>(ws + p.place);

  ProductArgs up{};
  up.x = static_cast<const uint8_t*>(x), up.x_scale = static_cast<const uint8_t*>(x_scale), up.order = order;
  up.w = static_cast<const uint8_t*>(gate_up), up.w_scale = static_cast<const uint8_t*>(gate_up_scale);
  up.tiles = tiles, up.tile_count = count;
  up.codes = ws + p.codes, up.scales = ws + p.scales;
  up.depth = (int32_t)dim, up.columns = (int32_t)(2 * inner), up.choices = (int32_t)choices;
  up.column_blocks = (int32_t)(inner / kBlock);
  ProductArgs dn{};
  dn.x = up.codes, dn.x_scale = up.scales, dn.order = order;
  dn.w = static_cast<const uint8_t*>(down), dn.w_scale = static_cast<const uint8_t*>(down_scale);
  dn.tiles = tiles, dn.tile_count = count;
  dn.y = reinterpret_cast<uint16_t*>(ws + p.y), dn.powers = ws + p.powers;
  dn.depth = (int32_t)inner, dn.columns = (int32_t)dim, dn.choices = (int32_t)choices;
  dn.column_blocks = (int32_t)((dim + 255) / 256);
  JoinArgs j{};
  j.ids = ids, j.place = place, j.weights = weights, j.y = dn.y, j.powers = dn.powers, j.out = out;
  j.choices = (int32_t)choices, j.first = (int32_t)first, j.experts = (int32_t)experts, j.dim = (int32_t)dim;
  j.groups_per_token = (int32_t)((dim / 8 + 255) / 256);
  DSA_CHECK_ARG(grid_fits(p.tiles * up.column_blocks + 7, 256) && grid_fits(p.tiles * dn.column_blocks + 7, 256) &&
                    grid_fits(tokens * j.groups_per_token, 256),
                "too many tokens for one launch");

  const GroupArgs group{ids, order, place, tiles, count, (int32_t)p.pairs, (int32_t)first, (int32_t)experts, 16 * p.rows};
  hipLaunchKernelGGL(group_pairs, dim3((unsigned)experts), dim3(kGroupThreads), 0, stream, group);
  DSA_CHECK_LAUNCH("grouping of pairs");
  if (const int status = launch_product<true>(up, p, stream)) return status;
  if (const int status = launch_product<false>(dn, p, stream)) return status;
  auto join = [&](auto kernel) {
    hipLaunchKernelGGL(kernel, dim3((unsigned)(tokens * j.groups_per_token)), dim3(256), 0, stream, j);
  };
  if (dtype == DSA_DTYPE_BF16) join(join_choices<Bf16Bits>);
  else if (dtype == DSA_DTYPE_F16) join(join_choices<_Float16>);
  else join(join_choices<float>);
  DSA_CHECK_LAUNCH("join of choices");
  return kOk;
}
