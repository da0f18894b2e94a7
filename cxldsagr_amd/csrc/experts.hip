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
// With so few pairs that an expert seldom has two, two launches: each pair by itself, and the
// token's results weighted and summed where they are formed.
// No atomics on values: results do not depend on the order of work-groups.
//
// The products run on v_mfma_scale_f32_*_f8f6f4, weights as the first operand, tokens as the
// second, so that a lane's results are of one token. The instruction multiplies by each
// operand's scale, a power of two per 32 values along K: the blocks of 128 cost nothing beyond
// that. Sums are in 32 bits, but for how the unit adds eight neighbouring products, in every form
// of its 8-bit instructions: each is cut (towards 0) to a multiple of 2^-13 of the largest's power
// of two. A product of 8 bits loses nothing down to 2^-6 of the largest, so that sums of normal
// values, 128 to 7,168 of them, are 1.4e-5 to 1.5e-5 of their size off: one in 700 codes of h falls
// on the other side of a border, and the result's error is 1.2 times that of products in 64 bits,
// 2.0e-3 of its size against 1.7e-3, most of it the rounding to bf16 (a row in which none of the
// largest codes moves has that alone; one row in 100 is 5e-3 off, the worst of 8,000 of 512 hidden
// values each 4e-2). 16-bit products, which lose nothing, need twice the unit's time and the codes'
// conversion: up's are of those in tiles of 32 rows and of pairs by themselves. Weights are laid out
// as waves read them (ExpertWeights), straight into registers: tiles of 16 rows by 128, 2 KB, in
// planes of 16 bytes a lane; tiles of gate and up in turn, so that a lane holds g and u of the
// same h; the rows of a wave's four tiles dealt out so that a lane's results are neighbours.
//
// What bounds it: reading the weights, up to some 100 rows an expert, where a kernel that only
// reads reaches 6.2 TB/s, past the caches 6.9 (32 experts of 7,168 by 2,048 dims, 8 choices: 1
// token 63 us, 5.6 TB/s; 64 tokens 232 us, 6.1; 128 experts, 128 tokens 860 us, 6.6); beyond that
// the matrix unit, which the card's power holds to 1.4 - 1.7 GHz (8,192 tokens 2,840 us, 2.03
// PFLOP/s: grouping 41, up 1,591, down 1,005, join 204, which is y's way to memory and back; the
// library's product of the same type 2.67. All of one card; another card's calls were within 4 %).
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

// Row tiles take the form of 32 rows of a weight by 32 tokens, 64 values deep: half as many
// instructions for the same work (one wave a SIMD issues the other in 45 clocks where the
// unit needs 32, this in 70 of 64).
template <int kW, int kX>
__device__ __forceinline__ v16f product32(v8i w, v8i x, v16f c, uint32_t w_scale, uint32_t x_scale) {
  return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(w, x, c, 0, 0, kW, (int)w_scale, kX, (int)x_scale);
}

// The same products in 16 bits, of codes that are converted for it: the unit adds these with 32
// bits throughout (sums of 7,168 are 1.2e-7 of their size off). They are up's where they cost
// little, while reading the weights is what takes time (1 token 64.1 -> 65.1 us, 64 tokens 249.6
// -> 251.1), and where a call has few values of h, with many rows of few experts at up to a fifth
// more (500 of one of 7,168 by 2,048 dims 56.4 -> 69.1). That is for a call's result as a whole, not
// for a row's, whose error in 8 bits is the same however many come with it: 1.4e-5 moves one code of
// h in 700 by a step, and where that is one of its row's largest, that row is up to 4e-2 of its size
// off. Of many such rows the result is 2.0e-3 off; of fewer than some 2^20 values a single one may
// be more of it than all other roundings (500 rows of one expert of 1,024 by 128 dims: 2.5e-3, in 16
// bits 1.7e-3; 250 rows of two of 8 of 4,096 by 2,048: 2.2e-3; 8,000 of 1,024 by 128: 1.9e-3).
// x takes both scales with it, 2^(a + b - 254) of their exponents' bytes, as the number whose
// exponent the conversion takes (255: NaN; products that bf16's exponents do not hold are far
// outside those of h).
__device__ __forceinline__ float both_scales(uint32_t a, uint32_t b) {
  const int e = min(max((int)(a + b) - 127, 0), 254);
  return __uint_as_float((a == 255 || b == 255 ? 255u : (uint32_t)e) << 23);
}
// Eight of a lane's 32 codes (part 0 .. 3) times that.
__device__ __forceinline__ v4u widened(v8i codes, int part, float scale) {
  v4u wide;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const uint32_t four = (uint32_t)codes[2 * part + i];
    wide[2 * i] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(four, scale, false));
    wide[2 * i + 1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(four, scale, true));
  }
  return wide;
}
__device__ __forceinline__ v4f wide_product(v4u w, v4u x, v4f c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(v8bf, w), __builtin_bit_cast(v8bf, x), c, 0, 0, 0);
}
__device__ __forceinline__ v16f wide_product(v4u w, v4u x, v16f c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(v8bf, w), __builtin_bit_cast(v8bf, x), c, 0, 0, 0);
}

// ------------------------------------------------------------ 1. groups --
// What every tile of an expert holds alike, so that a work-group finds its own in one look.
struct Tile {
  int32_t expert, row, rows;  // the expert's rows
  int32_t first, count;       // and its tiles
  int32_t unused[3];
};

struct GroupArgs {
  const int32_t* ids;   // [pairs]
  int32_t* tokens;      // [pairs]: the token of a row
  int32_t* place;       // [pairs]: the row of a pair (of this call's experts)
  Tile* tiles;
  int32_t* tile_count;
  int32_t pairs, choices, first, experts, tile_rows;
};

// Work-group e lists expert e's pairs. Each counts all experts' (in LDS), so that none waits
// for another: rows and tiles of the experts before e are sums over the counts. A wave takes
// a run of the pairs, so that a pair's row is the sum of what was found before it, kAtOnce of
// a lane's on their way at once: what bounds it is the way to memory and back (65,536 pairs
// of 32 experts with eight at once: 43 us).
template <int kAtOnce>
__global__ __launch_bounds__(kGroupThreads) void group_pairs(GroupArgs a) {
  // (Behind the last: pairs of other experts, a place for each lane, as one for all would
  // take them one after another.)
  __shared__ uint32_t counts[kMaxExperts + 64];
  __shared__ uint32_t of_wave[kGroupThreads / 64][3];
  const uint32_t expert = blockIdx.x, experts = a.experts;
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, waves = blockDim.x >> 6;
  constexpr int kPart = 64 * kAtOnce;
  const int run = ((a.pairs + waves - 1) / waves + 63) / 64 * 64;
  const int begin = wave * run < a.pairs ? wave * run : a.pairs, end = a.pairs - begin < run ? a.pairs : begin + run;
  // Experts of pairs base + lane, base + 64 + lane, ... (past the end: others).
  uint32_t e[kAtOnce];
  auto load = [&](int base) {
    int32_t id[kAtOnce];
#pragma unroll
    for (int i = 0; i < kAtOnce; ++i) {
      const int p = base + 64 * i + lane;
      id[i] = a.ids[p < end ? p : end - 1];
    }
#pragma unroll
    for (int i = 0; i < kAtOnce; ++i) {
      const uint32_t of = (uint32_t)id[i] - (uint32_t)a.first;
      e[i] = base + 64 * i + lane < end ? min(of, experts) : experts;
    }
  };
  if (begin < end) load(begin);
  for (uint32_t i = threadIdx.x; i < experts; i += blockDim.x) counts[i] = 0;
  __syncthreads();
  uint32_t found = 0;
  for (int base = begin; base < end; base += kPart) {
    if (base > begin) load(base);
#pragma unroll
    for (int i = 0; i < kAtOnce; ++i) {
      atomicAdd(&counts[e[i] < experts ? e[i] : experts + lane], 1u);
      found += e[i] == expert;
    }
  }
  found = sum_lanes(found);
  __syncthreads();
  // Rows and tiles of the experts before this one.
  uint32_t rows = 0, tiles = 0;
  for (uint32_t i = threadIdx.x; i < expert; i += blockDim.x)
    rows += counts[i], tiles += (counts[i] + a.tile_rows - 1) / a.tile_rows;
  rows = sum_lanes(rows), tiles = sum_lanes(tiles);
  if (lane == 0) of_wave[wave][0] = rows, of_wave[wave][1] = tiles, of_wave[wave][2] = found;
  __syncthreads();
  uint32_t row = 0, tile = 0, before = 0;
  for (int w = 0; w < waves; ++w) {
    row += of_wave[w][0], tile += of_wave[w][1];
    if (w < wave) before += of_wave[w][2];
  }
  const uint32_t own = counts[expert], own_tiles = (own + a.tile_rows - 1) / a.tile_rows;
  for (uint32_t t = threadIdx.x; t < own_tiles; t += blockDim.x)
    a.tiles[tile + t] = Tile{(int32_t)expert, (int32_t)row, (int32_t)own, (int32_t)tile, (int32_t)own_tiles, {}};
  if (expert == experts - 1 && threadIdx.x == 0) *a.tile_count = (int32_t)(tile + own_tiles);
  uint32_t next = row + before;
  for (int base = begin; base < end; base += kPart) {
    if (run > kPart) load(base);  // (else they are here still)
#pragma unroll
    for (int i = 0; i < kAtOnce; ++i) {
      const uint64_t all = __ballot(e[i] == expert);
      if (all == 0) continue;
      if (e[i] == expert) {
        const uint32_t to = next + (uint32_t)__popcll(all & ((1ull << lane) - 1));
        const int p = base + 64 * i + lane;
        a.tokens[to] = p / a.choices;
        a.place[p] = (int32_t)to;
      }
      next += (uint32_t)__popcll(all);
    }
  }
}

// ------------------------------------------------------ 2, 3. products --
struct ProductArgs {
  const uint8_t* x;        // rows of `depth` codes: tokens (up), pairs in order (down)
  const uint8_t* x_scale;  // [rows, depth / 128]
  const int32_t* tokens;   // up: of the rows
  const uint8_t* w;        // [experts][columns / 16][depth / 128][2048]
  const uint8_t* w_scale;  // [experts][columns / 128][depth / 128]
  const Tile* tiles;
  const int32_t* tile_count;
  uint8_t* codes;          // up: h [pairs, inner] and its scales
  uint8_t* scales;
  uint16_t* y;             // down: [pairs, columns] fp16, and its powers [pairs, columns / 64]
  uint8_t* powers;
  int32_t depth, columns, column_blocks;
};

__device__ __forceinline__ float silu(float g) {
  return g * __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(g * -kLog2E));
}

// h of kCount gates and ups of one row, and the largest magnitude's bits.
template <int kCount, typename Gate, typename Up>
__device__ __forceinline__ uint32_t hidden(float (&h)[kCount], Gate gate, Up up) {
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < kCount; ++i) {
    h[i] = silu(gate(i)) * up(i);
    const uint32_t bits = __float_as_uint(h[i]) & 0x7FFFFFFFu;
    top = top > bits ? top : bits;
  }
  return top;
}

// The power of two of 64 values of a row by their largest finite magnitude's bits: its
// exponent (at least 15: a smaller row of 64 keeps steps of 2^-136), and the factor that
// takes that magnitude to 2^14 .. 2^15.
struct Power {
  uint32_t exponent;
  float factor;
};
__device__ __forceinline__ Power power_of(uint32_t top) {
  const uint32_t e = (top >> 23) < 15u ? 15u : top >> 23;
  return Power{e, __uint_as_float((268u - e) << 23)};
}
__device__ __forceinline__ uint32_t finite_max(uint32_t top, float v) {
  const uint32_t bits = __float_as_uint(v) & 0x7FFFFFFFu;
  return bits < 0x7F800000u && bits > top ? bits : top;
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

// 16 bytes of a weight; kOnce: that no other work-group of the call wants, past the caches, of
// which the rest of the call has more then.
template <bool kOnce>
__device__ __forceinline__ v4u load_part(const v4u* from) {
  if constexpr (kOnce) return __builtin_nontemporal_load(from);
  return *from;
}

// Tile t of the wave's four, one step.
template <bool kOnce>
__device__ __forceinline__ v8i load_weight(const uint8_t* codes, int steps, int t, int s) {
  const v4u* from = reinterpret_cast<const v4u*>(codes + ((int64_t)t * steps + s) * kTile);
  return joined(load_part<kOnce>(from), load_part<kOnce>(from + 64));
}

// Row tiles: 32 kRows rows by 256 columns. Each wave keeps its 64 columns of the weight in
// registers, a step ahead; the rows' codes go into LDS straight from memory (two steps
// ahead, four buffers), where all four waves read them, an operand ahead of its products.
// Half-way through a step the waves meet: from there on the next step's rows may be read. A
// row's eight 16-byte parts are turned by its index, so that the rows' reads of one part fall
// on different banks.
// Rows' scales: up lays those of all steps out in LDS before the first; the scales of h come
// from memory a step ahead, where up has put them by tile.
// Per step of 128 a CU's matrix units take 256 kRows clocks, its LDS 160 kRows (four waves'
// reads and one write of 4 kRows KB at 128 bytes). Two work-groups of 128 rows a CU: one's
// start and end (11 and 8 of 144 thousand clocks of up, 6 and 9 of 51 of down) go on beside
// the other's products. 256 rows by four waves of twice the accumulators, or by eight waves,
// read a third less from L2 and were slower (8,192 tokens 2,890 and 3,170 us against 2,830);
// 96 rows were faster at 640 tokens of 32 experts alone (370 us against 387).
constexpr int kMaxSteps = 256;
// Steps of up whose rows' scales LDS holds (of 128 rows with two work-groups a CU).
constexpr int max_up_steps(int rows) { return rows <= 2 ? kMaxSteps : 124; }
template <int kRows, bool kUp>
struct TileLds {
  alignas(16) uint8_t rows[4][32 * kRows * kBlock];
  alignas(16) uint8_t scales[kUp ? max_up_steps(kRows) : 1][32][kRows];  // (a row's part of 32 last: one read holds all)
  alignas(4) uint8_t weight_scales[kUp ? max_up_steps(kRows) : kMaxSteps][2];
};

// The wave's weight tiles as two operands of 32 rows (up: gate's and up's), 64 deep: half k
// of a step. Lane (r, h): rows r of tiles `first` and `second`, bytes 32 h .. of the half.
template <bool kOnce>
__device__ __forceinline__ v8i load_weight32(const uint8_t* codes, int64_t tile, int k) {
  const v4u* from = reinterpret_cast<const v4u*>(codes + tile + k * 1024);
  return joined(load_part<kOnce>(from), load_part<kOnce>(from + 16));
}

// How a row's parts are turned: two rows and their eight parts are all 64 banks. 16 lanes are
// served at once, 0 .. 3 with 12 .. 15 and 20 .. 27, the other 16 of 32 together: eight of the
// first 16 rows and eight of the others, which must not fall on the same banks. (Turned by
// row % 8 alone half of the LDS's time went to conflicts.)
__device__ __forceinline__ uint32_t turn_of(uint32_t row) { return (row & 7) ^ (row >> 4 & 1); }

template <int kRows, bool kUp, bool kOnce>
__global__ __launch_bounds__(256, kRows == 1 ? 4 : kRows == 2 ? 3 : 2) void expert_product(ProductArgs a) {
  constexpr bool kWide = kUp && kRows == 1;  // products in 16 bits
  constexpr int kSize = 32 * kRows;  // rows of a tile
  __shared__ TileLds<kRows, kUp> lds;
  // Work-groups go round the eight XCDs: each takes a run of the work, in which an expert's
  // row tiles are neighbours and read the same columns of its weight through one L2.
  const uint32_t all = (uint32_t)(*a.tile_count * a.column_blocks), each = (all + 7) / 8;
  const uint32_t at = (blockIdx.x & 7) * each + (blockIdx.x >> 3);
  if ((blockIdx.x >> 3) >= each || at >= all) return;
  Tile tile = a.tiles[at / (uint32_t)a.column_blocks];
  const uint32_t within = at - (uint32_t)(tile.first * a.column_blocks);
  const int block = (int)(within / (uint32_t)tile.count), nth = (int)(within % (uint32_t)tile.count);
  const int tile_at = tile.first + nth;
  tile.row += nth * kSize;
  tile.rows = min(tile.rows - nth * kSize, kSize);

  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, r = lane & 31, h = lane >> 5;
  const int column = block * 256 + wave * kWaveCols;
  const int steps = a.depth / kBlock;
  const WaveWeight w = weight_of<kUp>(a, tile.expert, block, column, steps);
  // (weight_of gives the address of lane (g, r); here lanes 0 .. 15 and 16 .. 31 of a half
  // take rows of the operand's two tiles.)
  const int64_t tile_bytes = (int64_t)steps * kTile;
  const uint8_t* codes = w.codes - lane * 16 + (r >> 4) * (kUp ? 2 : 1) * tile_bytes + (h * 32 + (r & 15)) * 16;
  const int64_t second = (kUp ? 1 : 2) * tile_bytes;

  // This lane's parts of the rows that its wave fetches: 8 kRows rows, eight a load; and, of
  // up, the row whose scales this thread lays out, kPer threads a row. (Tokens' numbers first:
  // one way to memory and back for all.)
  constexpr int kLoads = kRows, kPer = 256 / kSize;
  auto row_of = [&](int in) -> int64_t {
    const int row = tile.row + min(in, tile.rows - 1);
    return kUp ? a.tokens[row] : row;
  };
  int64_t rows[kLoads];
#pragma unroll
  for (int i = 0; i < kLoads; ++i) rows[i] = row_of((wave * kLoads + i) * 8 + (lane >> 3));
  const int scale_row = threadIdx.x / kPer;
  const uint8_t* xs_row = kUp ? a.x_scale + row_of(scale_row) * steps : nullptr;
  uint64_t from[kLoads];
#pragma unroll
  for (int i = 0; i < kLoads; ++i)
    from[i] = (uint64_t)(a.x + rows[i] * a.depth + (((lane & 7) ^ turn_of((wave * kLoads + i) * 8 + (lane >> 3))) << 4));
  const uint32_t lds_rows = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint8_t*)&lds.rows[0][0];
  auto fetch = [&](int buffer, int i) {
    const uint32_t to = lds_rows + buffer * (kSize * kBlock) + (wave * kLoads + i) * 1024;
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off"
                 ::"s"(__builtin_amdgcn_readfirstlane(to)), "v"(from[i]) : "memory", "m0");
  };
  const uint32_t once = steps > 1 ? kBlock : 0;
#pragma unroll
  for (int i = 0; i < kLoads; ++i) fetch(0, i);
#pragma unroll
  for (int i = 0; i < kLoads; ++i) from[i] += once, fetch(1, i);
  v8i now[2][2];  // [half][operand]
#pragma unroll
  for (int i = 0; i < 4; ++i) now[i >> 1][i & 1] = load_weight32<kOnce>(codes, (i & 1) * second, i >> 1);

  // The weight's scales of all steps. (Down: of a block of 128 columns each pair of waves,
  // up: of gate and up.)
  {
    const WaveWeight one = weight_of<kUp>(a, tile.expert, block, block * 256, steps);
    const WaveWeight other = weight_of<kUp>(a, tile.expert, block, block * 256 + 128, steps);
    for (int s = threadIdx.x; s < steps; s += 256) {
      lds.weight_scales[s][0] = one.scale[0][s];
      lds.weight_scales[s][1] = (kUp ? one.scale[1] : other.scale[0])[s];
    }
  }
  if constexpr (kUp) {
    // The rows' scales of all steps, four at once where they are aligned.
    uint8_t* to = &lds.scales[0][scale_row & 31][scale_row >> 5];
    if ((steps & 3) == 0 && ((uintptr_t)a.x_scale & 3) == 0) {
      uint32_t four[max_up_steps(kRows) / 4 / kPer + 1];
      const int part = threadIdx.x % kPer;
#pragma unroll
      for (int i = 0; i < max_up_steps(kRows) / 4 / kPer + 1; ++i)
        if (4 * kPer * i < steps) {
          const int s = 4 * (kPer * i + part);
          four[i] = *reinterpret_cast<const uint32_t*>(xs_row + (s < steps ? s : 0));
        }
#pragma unroll
      for (int i = 0; i < max_up_steps(kRows) / 4 / kPer + 1; ++i) {
        const int s = 4 * (kPer * i + part);
        if (4 * kPer * i < steps && s < steps) {
#pragma unroll
          for (int k = 0; k < 4; ++k) to[(s + k) * kSize] = (uint8_t)(four[i] >> (8 * k));
        }
      }
    } else {
      for (int s = threadIdx.x % kPer; s < steps; s += kPer) to[s * kSize] = xs_row[s];
    }
  }
  // Down: this lane's rows' scales, of row r of all 32-row parts, a step every 32 kRows bytes.
  const uint8_t* row_scales = a.x_scale + (int64_t)tile_at * steps * kSize + r * kRows;
  wait_loads<0>();
  lds_barrier();

  // Part m, half k of a step: a lane's two 16-byte parts of row r are 4 k + 2 h and the next.
  const uint32_t lane_at = lds_rows + r * kBlock + (((2 * h) ^ turn_of(r)) << 4);
  // Operands in registers: the one ahead of the products, with the SIMD's other waves, hides
  // the LDS.
  constexpr int kRing = 2, kAhead = 1, kParts = 2 * kRows;
  v8i x[kRing];
  auto read = [&](uint32_t buffer, int q) {
    const uint32_t from = buffer * (kSize * kBlock) + (q % kRows) * 32 * kBlock;
    const uint32_t at = q < kRows ? lane_at : lane_at ^ 64;
    return joined(lds_load<v4u>(at + from), lds_load<v4u>((at ^ 16) + from));
  };
  using RowScales = std::conditional_t<kRows == 1, uint8_t, std::conditional_t<kRows == 2, uint16_t, uint32_t>>;
  auto scales_of = [&](int s) {
    const uint8_t* at = kUp ? &lds.scales[kUp ? s : 0][r][0] : row_scales + s * kSize;
    return (uint32_t)*reinterpret_cast<const RowScales*>(at);
  };
  auto weight_scales_of = [&](int s) {
    const uint32_t both = *reinterpret_cast<const uint16_t*>(&lds.weight_scales[s][0]);
    return kUp ? both : both >> (wave >> 1 << 3);
  };
#pragma unroll
  for (int q = 0; q < kAhead; ++q) x[q] = read(0, q);
  uint32_t xs = scales_of(0);
  uint32_t ws = weight_scales_of(0);

  v16f acc[kRows][2] = {};
#pragma unroll 1
  for (int s = 0; s < steps; ++s) {
    const int ahead = s + 1 < steps ? s + 1 : s;
    const uint32_t on = s + 2 < steps ? kBlock : 0;
    v8i next[2][2];
    uint32_t xs_next;
    uint32_t ws_next;
    static_for<kParts>([&](auto index) {
      constexpr int q = decltype(index)::value, m = q % kRows, k = q / kRows;
      __builtin_amdgcn_sched_barrier(0);
      // The next step's weight and scales and the rows of the one after are asked for in the
      // first half, behind the first products, which wait for this step's (what is asked for
      // before them would be waited for there), and a few at a time: a wave does not get on
      // while the path to L2 is full. (At the end the last rows come again, into buffers that
      // are not read.)
      if constexpr (q == 1) {
        xs_next = scales_of(ahead);
        ws_next = weight_scales_of(ahead);
      }
      constexpr int kOps = kLoads + 4, kPer = (kOps + kRows - 1) / kRows;
      if constexpr (q >= 1 && q <= kRows) {
        static_for<kPer>([&](auto which) {
          constexpr int op = (q - 1) * kPer + decltype(which)::value;
          // Rows and weights in turn while there are rows.
          constexpr bool fetches = op < 2 * kLoads && op % 2 == 0;
          constexpr int i = op < 2 * kLoads ? op / 2 : op - kLoads;
          if constexpr (fetches) from[i] += on, fetch((s + 2) & 3, i);
          else if constexpr (op < kOps) next[i >> 1][i & 1] = load_weight32<kOnce>(codes, (i & 1) * second + (int64_t)ahead * kTile, i >> 1);
        });
      }
      __builtin_amdgcn_sched_barrier(0);
      if constexpr (q == kRows) {
        // This wave's rows of the next step have come, and everyone's.
        wait_loads<kLoads + (kUp ? 8 : 9)>();
        __builtin_amdgcn_s_barrier();
        __builtin_amdgcn_sched_barrier(0);
      }
      x[(q + kAhead) % kRing] = q + kAhead < kParts ? read(s & 3, q + kAhead) : read((s + 1) & 3, q + kAhead - kParts);
      if constexpr (kWide) {
        const float scale[2] = {both_scales(xs >> (8 * m) & 255, ws & 255), both_scales(xs >> (8 * m) & 255, ws >> 8)};
        static_for<8>([&](auto part) {
          constexpr int o = decltype(part)::value & 1, i = decltype(part)::value / 2;
          acc[m][o] = wide_product(widened(now[k][o], i, 1.0f), widened(x[q % kRing], i, scale[o]), acc[m][o]);
        });
      } else {
        acc[m][0] = product32<0, m>(now[k][0], x[q % kRing], acc[m][0], ws, xs);
        acc[m][1] = product32<kUp ? 1 : 0, m>(now[k][1], x[q % kRing], acc[m][1], ws, xs);
      }
    });
#pragma unroll
    for (int i = 0; i < 4; ++i) now[i >> 1][i & 1] = next[i >> 1][i & 1];
    xs = xs_next;
    ws = ws_next;
  }
  // (What is still on its way into LDS has to land before the LDS is another's.)
  wait_loads<0>();

  // Lane (r, h) holds of row r the results 8 (i / 4) + 4 h + i % 4 of each operand: of the
  // tiles' dealt rows two runs, one for each p = (i / 4) % 2. Results go out through LDS, so
  // that an instruction writes whole lines (16 or 32 bytes of many rows at a time, a step's
  // time went by at each end). Parts of 16 bytes are turned by their row again.
  __syncthreads();
  if constexpr (kUp) {
    const int64_t inner = a.columns / 2;
    uint32_t* amax = reinterpret_cast<uint32_t*>(&lds.rows[0][0]);
    const uint32_t staged = lds_rows + 4 * kSize * sizeof(uint32_t);
    float hid[kRows][2][8];
#pragma unroll
    for (int m = 0; m < kRows; ++m) {
      uint32_t top = 0;
#pragma unroll
      for (int p = 0; p < 2; ++p) {
        const uint32_t of = hidden(hid[m][p], [&](int i) { return acc[m][0][(i >> 2) * 8 + p * 4 + (i & 3)]; },
                                   [&](int i) { return acc[m][1][(i >> 2) * 8 + p * 4 + (i & 3)]; });
        top = top > of ? top : of;
      }
      const auto both = __builtin_amdgcn_permlane32_swap(top, top, false, false);
      if (h == 0) amax[wave * kSize + m * 32 + r] = both[0] > both[1] ? both[0] : both[1];
    }
    __syncthreads();
#pragma unroll
    for (int m = 0; m < kRows; ++m) {
      const int in = m * 32 + r;
      uint32_t top = 0;
#pragma unroll
      for (int v = 0; v < 4; ++v) top = top > amax[v * kSize + in] ? top : amax[v * kSize + in];
      const float scale = scale_from_amax_bits(top, true);
#pragma unroll
      for (int p = 0; p < 2; ++p) {
        v2u out;
        uint32_t lo, hi;
        quantize_eight(hid[m][p], scale, true, lo, hi);
        out[0] = lo, out[1] = hi;
        lds_store(staged + in * kBlock + (((wave * 2 + p) ^ (in & 7)) << 4) + 8 * h, out);
      }
      if (wave == 0 && h == 0 && in < tile.rows)
        a.scales[((int64_t)tile_at * (inner / kBlock) + block) * kSize + r * kRows + m] = (uint8_t)(__float_as_uint(scale) >> 23);
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kRows; ++i) {
      const int row = i * 32 + wave * 8 + (lane >> 3), part = lane & 7;
      const v4u out = lds_load<v4u>(staged + row * kBlock + ((part ^ (row & 7)) << 4));
      if (row < tile.rows) *reinterpret_cast<v4u*>(a.codes + (tile.row + row) * inner + block * kBlock + part * 16) = out;
    }
  } else {
#pragma unroll
    for (int m = 0; m < kRows; ++m) {
      const int in = m * 32 + r;
      uint32_t top = 0;
#pragma unroll
      for (int i = 0; i < 32; ++i) top = finite_max(top, acc[m][i >> 4][i & 15]);
      const auto both = __builtin_amdgcn_permlane32_swap(top, top, false, false);
      const Power power = power_of(both[0] > both[1] ? both[0] : both[1]);
#pragma unroll
      for (int p = 0; p < 2; ++p)
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          // Eight neighbours: columns 32 p + 16 h + 8 half .. of the wave's 64.
          v4u out;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int at = 8 * half + 2 * i, of = (at >> 2 & 1) * 8 + p * 4 + (at & 3);
            out[i] = F16::pack(acc[m][at >> 3][of] * power.factor, acc[m][at >> 3][of + 1] * power.factor);
          }
          lds_store(lds_rows + in * 512 + (((wave * 8 + 4 * p + 2 * h + half) ^ r) << 4), out);
        }
      if (h == 0 && column < a.columns && in < tile.rows)
        a.powers[(tile.row + in) * (int64_t)(a.columns / kWaveCols) + column / kWaveCols] = (uint8_t)power.exponent;
    }
    __syncthreads();
    const int part = lane & 31;
#pragma unroll
    for (int i = 0; i < kSize / 8; ++i) {
      const int row = i * 8 + wave * 2 + (lane >> 5);
      const v4u out = lds_load<v4u>(lds_rows + row * 512 + ((part ^ (row & 31)) << 4));
      if (row < tile.rows && block * 256 + part * 8 < a.columns)
        *reinterpret_cast<v4u*>(a.y + (tile.row + row) * (int64_t)a.columns + block * 256 + part * 8) = out;
    }
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
  // (All loads of a few choices are on their way before the first is used.)
  constexpr int kAtOnce = 8;
  for (int c0 = 0; c0 < a.choices; c0 += kAtOnce) {
    v8hf y[kAtOnce];
    float weight[kAtOnce];
    uint32_t power[kAtOnce];
    bool here[kAtOnce];
#pragma unroll
    for (int i = 0; i < kAtOnce; ++i) {
      const int c = c0 + i < a.choices ? c0 + i : a.choices - 1;
      const int64_t pair = token * a.choices + c;
      here[i] = c0 + i < a.choices && (uint32_t)a.ids[pair] - (uint32_t)a.first < (uint32_t)a.experts;
      weight[i] = a.weights[pair];
      if (here[i]) {
        const int64_t row = a.place[pair];
        // (Past the caches: 8,192 tokens 226 - 233 -> 201 - 209 us of this launch, less than the
        // whole call varies by; 2,048 53 -> 51, 64 5.0 both.)
        y[i] = __builtin_bit_cast(v8hf, __builtin_nontemporal_load(reinterpret_cast<const v4u*>(a.y + row * a.dim + column)));
        power[i] = a.powers[row * (a.dim / kWaveCols) + column / kWaveCols];
      }
    }
#pragma unroll
    for (int i = 0; i < kAtOnce; ++i) {
      if (!here[i]) continue;
      const float unit = __uint_as_float((power[i] - 14u) << 23);
#pragma unroll
      for (int j = 0; j < 8; ++j) sum[j] += (float)y[i][j] * unit * weight[i];
    }
  }
  Eight out;
#pragma unroll
  for (int i = 0; i < 8; ++i) out.v[i] = rounded<T>(sum[i]);
  *reinterpret_cast<Eight*>(static_cast<T*>(a.out) + token * a.dim + column) = out;
}

// ------------------------------------------------------------- one by one --
// With so few tokens that an expert seldom has two, each pair by itself: no groups, and the
// results weighted and summed where they are formed. Two launches instead of four.
struct PairArgs {
  const uint8_t* x;
  const uint8_t* x_scale;
  const int32_t* ids;
  const float* weights;
  const uint8_t* w;        // gate and up; down
  const uint8_t* w_scale;
  float* hidden;           // [pairs, inner]
  void* out;
  int32_t dim, inner, choices, first, experts, blocks, parts;
};

// What a wave's products of one step need: 64 rows of a weight, a token's codes, their scales.
struct Step {
  v8i w[4], x;
  uint32_t w_scale[2], x_scale;
};

// up: a work-group takes 32 columns of h, a quarter of the depth a wave, three steps at once
// (what bounds it is reading the weight: 8 KB a step, of which a CU wants some 40 under way).
template <bool kOnce>
__global__ __launch_bounds__(256, 2) void pair_hidden(PairArgs a) {
  constexpr int kDepth = 3;
  __shared__ float part[4][4][16];
  const int pair = blockIdx.x / a.blocks, block = blockIdx.x % a.blocks;
  const uint32_t expert = (uint32_t)a.ids[pair] - (uint32_t)a.first;
  if (expert >= (uint32_t)a.experts) return;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, g = lane >> 4;
  const int steps = a.dim / kBlock, begin = steps * wave / 4, end = steps * (wave + 1) / 4;
  const int64_t token = pair / a.choices;
  const uint8_t* w = a.w + ((int64_t)expert * (a.inner / 8) + block * 4) * steps * kTile + lane * 16;
  const uint8_t* gate = a.w_scale + ((int64_t)expert * (a.inner / 64) + block / 4) * steps;
  const uint8_t* up = gate + (int64_t)(a.inner / kBlock) * steps;
  const uint8_t* x = a.x + token * a.dim + g * 16;
  const uint8_t* xs = a.x_scale + token * steps;
  Step ring[kDepth];
  auto load = [&](Step& to, int s) {
#pragma unroll
    for (int t = 0; t < 4; ++t) to.w[t] = load_weight<kOnce>(w, steps, t, s);
    to.w_scale[0] = gate[s], to.w_scale[1] = up[s];
    const v4u* from = reinterpret_cast<const v4u*>(x + s * kBlock);
    to.x = joined(from[0], from[4]);
    to.x_scale = xs[s];
  };
  v4f acc[4] = {};
  if (begin < end) {
#pragma unroll
    for (int d = 0; d < kDepth; ++d) load(ring[d], begin + d < end ? begin + d : end - 1);
    auto multiply = [&](const Step& of) {
      const float scale[2] = {both_scales(of.x_scale, of.w_scale[0]), both_scales(of.x_scale, of.w_scale[1])};
#pragma unroll
      for (int part = 0; part < 4; ++part) {
        // (x with the scales of gate's tiles and of up's)
        const v4u wide[2] = {widened(of.x, part, scale[0]), widened(of.x, part, scale[1])};
#pragma unroll
        for (int t = 0; t < 4; ++t) acc[t] = wide_product(widened(of.w[t], part, 1.0f), wide[t & 1], acc[t]);
      }
    };
    int s = begin;
    for (; s + kDepth <= end; s += kDepth) {
#pragma unroll
      for (int d = 0; d < kDepth; ++d) {
        multiply(ring[d]);
        load(ring[d], s + d + kDepth < end ? s + d + kDepth : end - 1);
      }
    }
#pragma unroll
    for (int d = 0; d < kDepth - 1; ++d)
      if (s + d < end) multiply(ring[d]);
  }
  // (All 16 columns of the product are the token's.)
  if ((lane & 15) == 0) {
#pragma unroll
    for (int t = 0; t < 4; ++t) *reinterpret_cast<v4f*>(&part[wave][t][4 * g]) = acc[t];
  }
  __syncthreads();
  const int c = threadIdx.x;  // column 8 g + 4 j + i of h: results 4 g + i of the tiles 2 j and 2 j + 1
  if (c >= 32) return;
  const int j = c >> 2 & 1, at = c >> 3 << 2 | (c & 3);
  float gated = 0.0f, upped = 0.0f;
#pragma unroll
  for (int v = 0; v < 4; ++v) gated += part[v][2 * j][at], upped += part[v][2 * j + 1][at];
  a.hidden[(int64_t)pair * a.inner + block * 32 + c] = silu(gated) * upped;
}

// down: a work-group takes a token's 32 columns: while the first weights are on their way
// it forms the codes of all choices' h, then a wave takes a choice's part of the depth after
// another: the products, and the weight.
constexpr int kPairCodes = 65536;
template <typename T, bool kOnce>
__global__ __launch_bounds__(1024) void pair_result(PairArgs a) {
  constexpr int kDepth = 4;
  __shared__ __align__(16) uint8_t codes[kPairCodes];
  __shared__ uint8_t scales[kPairCodes / kBlock];
  __shared__ float part[16][2][16];
  const int64_t token = blockIdx.x / a.blocks;
  const int block = blockIdx.x % a.blocks;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, g = lane >> 4;
  const int steps = a.inner / kBlock, units = a.choices * a.parts, waves = blockDim.x >> 6;
  struct {
    v8i w[2];
    uint32_t scale;
  } ring[kDepth];
  const uint8_t* w = nullptr;
  const uint8_t* ws = nullptr;
  auto load = [&](auto& to, int s) {
#pragma unroll
    for (int t = 0; t < 2; ++t) to.w[t] = load_weight<kOnce>(w, steps, t, s);
    to.scale = ws[s];
  };
  // The choices that are here, a bit each (64 at most).
  const uint32_t mine = lane < a.choices ? (uint32_t)a.ids[token * a.choices + lane] - (uint32_t)a.first : ~0u;
  const uint64_t here = __ballot(mine < (uint32_t)a.experts);
  // A unit's expert (past the last: none) and its first weights.
  int begin = 0, end = 0;
  auto start = [&](int u) {
    if (u >= units) return false;
    const uint32_t expert = (uint32_t)a.ids[token * a.choices + u / a.parts] - (uint32_t)a.first;
    if (expert >= (uint32_t)a.experts) return false;
    const int at = u % a.parts;
    begin = steps * at / a.parts, end = steps * (at + 1) / a.parts;
    w = a.w + ((int64_t)expert * (a.dim / 16) + block * 2) * steps * kTile + lane * 16;
    ws = a.w_scale + ((int64_t)expert * (a.dim / kBlock) + block / 4) * steps;
#pragma unroll
    for (int d = 0; d < kDepth; ++d) load(ring[d], begin + d < end ? begin + d : end - 1);
    return true;
  };
  bool some = start(wave);

  // 16 lanes a block of 128. (Of choices that are not here nothing was written.)
  for (int i = threadIdx.x >> 4; i < a.choices * steps; i += blockDim.x >> 4) {
    if (!(here >> (i / steps) & 1)) continue;
    const float4* from = reinterpret_cast<const float4*>(a.hidden + token * a.choices * a.inner + i * kBlock + (threadIdx.x & 15) * 8);
    const float4 one = from[0], two = from[1];
    const float v[8] = {one.x, one.y, one.z, one.w, two.x, two.y, two.z, two.w};
    uint32_t top = 0, lo, hi;
#pragma unroll
    for (int j = 0; j < 8; ++j) top = max(top, __float_as_uint(v[j]) & 0x7FFFFFFFu);
    const float scale = scale_from_amax_bits(max_abs_bits_reduce<16>(top), true);
    quantize_eight(v, scale, true, lo, hi);
    *reinterpret_cast<uint2*>(&codes[i * kBlock + (threadIdx.x & 15) * 8]) = make_uint2(lo, hi);
    if ((threadIdx.x & 15) == 0) scales[i] = (uint8_t)(__float_as_uint(scale) >> 23);
  }
  __syncthreads();

  v4f total[2] = {};
  for (int u = wave; u < units; u += waves) {
    if (u > wave) some = start(u);
    if (!some) continue;
    const int choice = u / a.parts;
    v4f acc[2] = {};
    for (int s = begin; s < end; s += kDepth) {
#pragma unroll
      for (int d = 0; d < kDepth; ++d) {
        if (s + d >= end) break;
        const v4u* x = reinterpret_cast<const v4u*>(&codes[(choice * steps + s + d) * kBlock + g * 16]);
        const v8i of = joined(x[0], x[4]);
        const uint32_t x_scale = scales[choice * steps + s + d];
#pragma unroll
        for (int t = 0; t < 2; ++t) acc[t] = product(ring[d].w[t], of, acc[t], ring[d].scale, x_scale);
        load(ring[d], s + d + kDepth < end ? s + d + kDepth : end - 1);
      }
    }
    const float weight = a.weights[token * a.choices + choice];
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i) total[t][i] += acc[t][i] * weight;
  }
  if ((lane & 15) == 0) {
#pragma unroll
    for (int t = 0; t < 2; ++t) *reinterpret_cast<v4f*>(&part[wave][t][4 * g]) = total[t];
  }
  __syncthreads();
  const int c = threadIdx.x;  // result 4 g + i of tile t: column 16 g + 4 t + i of 64, t 0 and 1 or 2 and 3
  if (c >= 32) return;
  const int t = c >> 2 & 1, at = c >> 3 << 2 | (c & 3);
  float sum = 0.0f;
  for (int v = 0; v < waves; ++v) sum += part[v][t][at];
  static_cast<T*>(a.out)[token * a.dim + block / 2 * 64 + (c >> 3) * 16 + (block & 1) * 8 + t * 4 + (c & 3)] = rounded<T>(sum);
}

// ----------------------------------------------------------------- calls --
struct Plan {
  int64_t pairs, tiles;       // of the longest call, and its row tiles at most
  int rows;                   // 32-row parts of a tile; 0: each pair by itself
  int parts;                  // of the depth of a pair's down
  bool once;                  // whether a weight is read by one work-group, seldom by more
  // Offsets of the workspace's parts.
  int64_t count, list, tokens, place, codes, scales, y, powers, bytes;
};

Plan plan_of(int64_t tokens, int64_t choices, int64_t dim, int64_t inner, int64_t experts, int64_t total) {
  Plan p{};
  p.pairs = tokens * choices;
  // Pair by pair up to three quarters as many pairs as experts, where a token's codes fit into
  // LDS and the weights of the pairs that are to be expected here stay below 500 MB: beyond that
  // tiles fill the card and read what two pairs share once (8 choices of 7,168 by 2,048 dims, 44
  // MB a pair; pairs by themselves and in tiles: 32 experts 1 token 65 us against 99, 2 tokens 120
  // against 111; 256 experts 1 token 74 against 101, 12 681 against 558, 24 1,337 against 912; 32 of
  // 256 here 10 tokens 95 against 103, 12 117 against 111, 24 202 against 143. 6 of 64 experts of
  // 2,048 by 1,408: 6 tokens 57 against 58, 8 68 against 68).
  const int64_t few = total * 3 / 4 > choices ? total * 3 / 4 : choices;
  const double weights = (double)p.pairs * experts / total * (3.0 * dim * inner);
  if (p.pairs <= few && weights <= 5e8 && choices * inner <= kPairCodes && grid_fits(p.pairs * (inner / 32), 256) &&
      grid_fits(tokens * (dim / 32), 1024)) {
    p.parts = (int)(choices >= 16 ? 1 : 16 / choices);
    if (p.parts > inner / kBlock) p.parts = (int)(inner / kBlock);
    p.bytes = p.pairs * inner * 4;
    // One token's choices are of different experts, few pairs' seldom the same (8 experts a token,
    // 32 of 7,168 by 2,048 dims here: 1 token 66.9 -> 63.5 us, 8 of 256 in all 85.7 -> 82.3; 16
    // would be 129.6 -> 136.6).
    p.once = tokens == 1 || p.pairs * 4 <= total;
    return p;
  }
  // Rows of an expert, on average: tiles that most experts fill once, as long as reading the
  // weights is what takes time (32 experts of 7,168 by 2,048 dims: 16 rows 250, 251, 254 us in
  // tiles of 32, 64, 128; 24 rows 274, 253, 258; 48 rows 287, 261, 267; 64 rows 338, 301, 274).
  const int64_t mean = p.pairs / total;
  p.rows = mean <= 16 ? 1 : mean <= 48 ? 2 : 4;
  if (dim > max_up_steps(4) * kBlock && p.rows > 2) p.rows = 2;
  // Few values of h (of the pairs that are to be expected here) want 16-bit products, for the
  // result as a whole (above wide_product). (In tiles of 64
  // rows these took longer, with half as many work-groups: 250 tokens, 2 of 2 experts of
  // 4,096 by 2,048 dims, one here, 44.6 -> 53.7 us, 90 tokens, 6 of 16 of 4,096 by 512, 55.1 -> 63.6.)
  if (p.pairs * experts / total * inner <= 1 << 20) p.rows = 1;
  // Most experts have one tile, whose columns are one work-group's (32 experts of 7,168 by 2,048
  // dims: 12 rows 250 -> 232 us, 40 262 -> 239, 88 294 -> 266; 120 354 -> 350, 160 would be 402 ->
  // 503; 16 of 4,096 by 1,408, 40 rows in tiles of 32, 77.8 -> 79.4).
  p.once = mean * 4 <= 3 * 32 * p.rows;
  const int64_t size = 32 * p.rows;
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
  p.tokens = part(p.pairs * 4);
  p.place = part(p.pairs * 4);
  p.codes = part(p.pairs * inner);
  p.scales = part(p.tiles * size * (inner / kBlock));  // (of whole tiles)
  p.y = part(p.pairs * dim * 2);
  p.powers = part(p.pairs * (dim / kWaveCols));
  p.bytes = at;
  return p;
}

// Work-groups of a product: up's tiles times 128 hidden columns, down's times 256 of the result.
int64_t up_blocks(int64_t inner) { return inner / kBlock; }
int64_t down_blocks(int64_t dim) { return (dim + 255) / 256; }

int check_shape(int64_t tokens, int64_t choices, int64_t dim, int64_t inner, int64_t experts, int64_t total) {
  DSA_CHECK_ARG(dim >= kBlock && dim % kBlock == 0 && dim <= 32768 && inner >= kBlock && inner % kBlock == 0 &&
                    inner <= 32768,
                "dims must be whole blocks of 128, 32768 at most");
  DSA_CHECK_ARG(experts >= 1 && experts <= kMaxExperts && total >= experts && total <= (1 << 30),
                "experts must number 1 to %d, total at least as many and at most 2^30", kMaxExperts);
  DSA_CHECK_ARG(choices >= 1 && choices <= 64, "choices must number 1 to 64");
  DSA_CHECK_ARG(tokens >= 0 && tokens <= (1 << 22), "tokens must number 0 to 2^22");
  // (Here, so that the size's query refuses what the call would.)
  const int64_t tiles = plan_of(tokens, choices, dim, inner, experts, total).tiles;
  DSA_CHECK_ARG(grid_fits(tiles * up_blocks(inner) + 7, 256) && grid_fits(tiles * down_blocks(dim) + 7, 256),
                "too many tokens for one launch");
  return kOk;
}

template <bool kUp>
int launch_product(const ProductArgs& a, const Plan& p, hipStream_t stream) {
  auto go = [&](auto kernel, int64_t groups) {
    hipLaunchKernelGGL(kernel, dim3((unsigned)groups), dim3(256), 0, stream, a);
  };
  const int64_t groups = (p.tiles * a.column_blocks + 7) / 8 * 8;
  auto pick = [&](auto once) {
    constexpr bool kOnce = decltype(once)::value;
    if (p.rows == 1) go(expert_product<1, kUp, kOnce>, groups);
    else if (p.rows == 2) go(expert_product<2, kUp, kOnce>, groups);
    else go(expert_product<4, kUp, kOnce>, groups);
  };
  if (p.once) pick(std::true_type{});
  else pick(std::false_type{});
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
  if (p.rows == 0) {
    PairArgs one{};
    one.x = static_cast<const uint8_t*>(x), one.x_scale = static_cast<const uint8_t*>(x_scale);
    one.ids = ids, one.weights = weights, one.hidden = static_cast<float*>(workspace), one.out = out;
    one.dim = (int32_t)dim, one.inner = (int32_t)inner, one.choices = (int32_t)choices;
    one.first = (int32_t)first, one.experts = (int32_t)experts, one.parts = p.parts;
    one.w = static_cast<const uint8_t*>(gate_up), one.w_scale = static_cast<const uint8_t*>(gate_up_scale);
    one.blocks = (int32_t)(inner / 32);
    auto up = [&](auto kernel) {
      hipLaunchKernelGGL(kernel, dim3((unsigned)(p.pairs * one.blocks)), dim3(256), 0, stream, one);
    };
    if (p.once) up(pair_hidden<true>);
    else up(pair_hidden<false>);
    DSA_CHECK_LAUNCH("hidden values of pairs");
    one.w = static_cast<const uint8_t*>(down), one.w_scale = static_cast<const uint8_t*>(down_scale);
    one.blocks = (int32_t)(dim / 32);
    const int units = (int)choices * p.parts, threads = 64 * (units < 16 ? units : 16);
    auto go = [&](auto kernel) {
      hipLaunchKernelGGL(kernel, dim3((unsigned)(tokens * one.blocks)), dim3(threads), 0, stream, one);
    };
    auto pick = [&](auto once) {
      constexpr bool kOnce = decltype(once)::value;
      if (dtype == DSA_DTYPE_BF16) go(pair_result<Bf16Bits, kOnce>);
      else if (dtype == DSA_DTYPE_F16) go(pair_result<_Float16, kOnce>);
      else go(pair_result<float, kOnce>);
    };
    if (p.once) pick(std::true_type{});
    else pick(std::false_type{});
    DSA_CHECK_LAUNCH("results of pairs");
    return kOk;
  }
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  Tile* tiles = reinterpret_cast<Tile*>(ws + p.list);
  int32_t* count = reinterpret_cast<int32_t*>(ws + p.count);
  int32_t* row_tokens = reinterpret_cast<int32_t*>(ws + p.tokens);
  int32_t* place = reinterpret_cast<int32_t*>(ws + p.place);

  ProductArgs up{};
  up.x = static_cast<const uint8_t*>(x), up.x_scale = static_cast<const uint8_t*>(x_scale), up.tokens = row_tokens;
  up.w = static_cast<const uint8_t*>(gate_up), up.w_scale = static_cast<const uint8_t*>(gate_up_scale);
  up.tiles = tiles, up.tile_count = count;
  up.codes = ws + p.codes, up.scales = ws + p.scales;
  up.depth = (int32_t)dim, up.columns = (int32_t)(2 * inner);
  up.column_blocks = (int32_t)up_blocks(inner);
  ProductArgs dn{};
  dn.x = up.codes, dn.x_scale = up.scales;
  dn.w = static_cast<const uint8_t*>(down), dn.w_scale = static_cast<const uint8_t*>(down_scale);
  dn.tiles = tiles, dn.tile_count = count;
  dn.y = reinterpret_cast<uint16_t*>(ws + p.y), dn.powers = ws + p.powers;
  dn.depth = (int32_t)inner, dn.columns = (int32_t)dim;
  dn.column_blocks = (int32_t)down_blocks(dim);
  JoinArgs j{};
  j.ids = ids, j.place = place, j.weights = weights, j.y = dn.y, j.powers = dn.powers, j.out = out;
  j.choices = (int32_t)choices, j.first = (int32_t)first, j.experts = (int32_t)experts, j.dim = (int32_t)dim;
  j.groups_per_token = (int32_t)((dim / 8 + 255) / 256);

  const GroupArgs group{ids, row_tokens, place, tiles, count, (int32_t)p.pairs, (int32_t)choices, (int32_t)first,
                        (int32_t)experts, 32 * p.rows};
  // (A wave for every 256 pairs, up to 16: with fewer the work-groups start and meet sooner.)
  const int64_t waves = (p.pairs + 255) / 256;
  auto list = [&](auto kernel) {
    hipLaunchKernelGGL(kernel, dim3((unsigned)experts), dim3((unsigned)(waves < 16 ? 64 * waves : (int64_t)kGroupThreads)), 0,
                       stream, group);
  };
  if (waves <= 16) list(group_pairs<4>);
  else if (waves <= 32) list(group_pairs<8>);
  else list(group_pairs<32>);
  DSA_CHECK_LAUNCH("grouping of pairs");
  if (const int status = launch_product<true>(up, p, stream)) return status;
  if (const int status = launch_product<false>(dn, p, stream)) return status;
  // (A launch holds 2^24 - 1 work-groups; the tokens behind take another.)
  const int64_t at_once = ((1ll << 24) - 1) / j.groups_per_token, out_bytes = dim * (dtype == DSA_DTYPE_F32 ? 4 : 2);
  auto join = [&](auto kernel) {
    for (int64_t begin = 0; begin < tokens; begin += at_once) {
      const int64_t some = tokens - begin < at_once ? tokens - begin : at_once;
      JoinArgs of = j;
      of.ids += begin * choices, of.place += begin * choices, of.weights += begin * choices;
      of.out = static_cast<uint8_t*>(out) + begin * out_bytes;
      hipLaunchKernelGGL(kernel, dim3((unsigned)(some * j.groups_per_token)), dim3(256), 0, stream, of);
    }
  };
  if (dtype == DSA_DTYPE_BF16) join(join_choices<Bf16Bits>);
  else if (dtype == DSA_DTYPE_F16) join(join_choices<_Float16>);
  else join(join_choices<float>);
  DSA_CHECK_LAUNCH("join of choices");
  return kOk;
}
