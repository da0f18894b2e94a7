// Causal attention over packed sequences with grouped heads, forward.
//
// Per sequence of n_q queries and n_k keys, head h of H reading KV head
// h / G (G = H / H_kv): out = softmax(scale q k^T) v over the keys
// j <= i + n_k - n_q of query i (causal; every key otherwise), in fp32 from
// 16-bit inputs, probabilities rounded to 16 bits before the product with V;
// a query without a visible key gives zeros. 2 (d_qk + d_v) flop per pair.
//
// Mapping (gfx950, wave64). The G heads that share a KV head are rows of one problem:
// row r of a sequence is token r / G, head r % G, so that single tokens of grouped
// heads fill a tile and K and V are staged once for all of them. A work-group has 128
// rows, 32 per wave, two work-groups share a CU (one's start, masks and stores run
// beside the other's products; 256 rows of one work-group took 285 us where these take
// 185: 2,048 tokens, 128 heads of 192 / 128), and walks the keys in stages of 32. A
// wave computes S^T = K Q^T (v_mfma_f32_32x32x16, Q^T in registers). The result's layout
// - a lane holds 16 keys of one row - is the operand layout of O^T += V^T P^T once the
// keys of V^T are read in the same order, so probabilities never leave registers and a
// row's softmax state and rescale factor belong to its lane.
// Software pipeline: the products S of a stage run beside the softmax of the stage
// before, then that stage's product with V beside the maxima of the new one.
//
// What bounds it: in long calls the matrix unit at the clock that the power limit leaves
// (1.84 GHz in the call above, 928 TFLOP/s) and its starts and ends; 8,192 tokens reach 1.0
// PFLOP/s, where a library product of large matrices reaches 1.36. In batches of short
// sequences the start and end of a work-group, 9k to 15k cycles (7 prompts of 4,001 tokens,
// 37 us); with few rows the loads of K and V (8 single tokens over 40,000 keys, 30 us and 4
// for the join, 4.9 TB/s). One cut serves a whole call: a prompt of 2,048 tokens beside one
// token over 40,000 keys (32 heads on 8 of 128 dims) takes 672 us, apart 55 and 35.
// Q loads and stores in pieces of 64 bytes, by lanes trading, took as long as they save.
//
// Stages arrive by LDS DMA two ahead, in blocks of 16 rows by 64 bytes: lane l brings
// chunk (l % 4) ^ (l / 16) (16 bytes) of row l / 4, which makes global reads whole
// 64-byte segments and both the K reads (16 rows, one chunk) and the transposing V
// reads (4 rows, 4 chunks) free of bank conflicts.
#include "attention_core.h"
#include "../../include/dsa_gfx950.h"

namespace dsa {
namespace {

// Keys of a stage.
constexpr int kStageKeys = 32;

// How a kernel is cut: kWaves waves of 32 rows; a stage's loads are issued kDistance
// stages before it is entered. K of a stage is read until the next is entered, V for
// two stages more.
template <int kWaves_, int kDistance_>
struct Cut {
  static constexpr int kWaves = kWaves_, kDistance = kDistance_;
  static constexpr int kRows = 32 * kWaves, kThreads = 64 * kWaves;
  static constexpr int kBufK = kDistance + 1, kBufV = kDistance + 3;
};

struct PromptArgs {
  const uint16_t* q;
  const uint16_t* k;
  const uint16_t* v;
  uint16_t* out;
  float* parts;    // [splits][q_tokens * heads][d_v], splits > 1 only
  float2* stats;   // [splits][q_tokens * heads]
  int64_t q_token, q_head, k_token, k_head, v_token, v_head;  // strides, elements
  int32_t heads, split_stages, causal, ranked;
  float scale_log2;
};

// The row tile of a rank among all tiles of up to 64 sequences by the stages of keys
// that their last row sees, most first: lane b looks at sequence b, of n_q queries and
// n_k keys (0 of both past the last), less than 2^16 tiles in all. The tiles of a
// sequence see more the later they are, so the tiles that see more than x stages are
// counted in closed form, a search over x, four at a time, finds how many the rank's
// tile sees, and a scan which of the tiles that see as many it is. Neighbours are then of
// different sequences; without it a batch's longest sequences start when others have
// run. See prompt_plan for where it is used. `which` is -1 past the last tile.
template <int kTileRows>
__device__ __forceinline__ void tile_of_rank(int rank, uint32_t group, int causal, int n_q, int n_k, int& which,
                                             uint32_t& tile_row) {
  const int history = n_k - n_q;
  const int tiles = (int)(((uint32_t)n_q * group + kTileRows - 1) / kTileRows);
  // This lane's tiles that see more than x stages (x = -1: all).
  auto above = [&](int x) -> uint32_t {
    const int keys = x * kStageKeys;
    const int y = causal ? keys - history : 0;  // of its last row's token at least
    const int more = y <= 0 ? tiles : max(tiles - (int)((uint32_t)y * group / kTileRows), 0);
    return x < 0 ? tiles : keys >= n_k ? 0 : more;
  };
  auto first = [](uint32_t v) -> int { return __builtin_amdgcn_readfirstlane((int)v); };
  const int all = first(sum_lanes(tiles));
  // The smallest x that at most `rank` tiles see more than.
  int lo = -1, hi = (first(max_lanes((uint32_t)n_k)) + kStageKeys - 1) / kStageKeys;
  which = -1;
  if (rank >= all) return;
  while (hi - lo > 1) {
    const int step = (hi - lo + 4) / 5;
    int x[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = min(lo + (i + 1) * step, hi);
    const uint32_t low = first(sum_lanes(above(x[0]) | above(x[1]) << 16));
    const uint32_t high = first(sum_lanes(above(x[2]) | above(x[3]) << 16));
    const int counts[4] = {(int)(low & 0xFFFF), (int)(low >> 16), (int)(high & 0xFFFF), (int)(high >> 16)};
    int below = lo;
#pragma unroll
    for (int i = 3; i >= 0; --i)
      if (counts[i] <= rank) hi = x[i];
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (counts[i] > rank) below = x[i];
    lo = below;
  }
  const int more = above(hi), same = above(hi - 1) - more;
  const int place = rank - first(sum_lanes(more)) - (int)sum_below((uint32_t)same);
  const uint64_t mine = __builtin_amdgcn_ballot_w64(place >= 0 && place < same);
  if (mine == 0) return;
  which = __builtin_ctzll(mine);
  const int tile = __builtin_amdgcn_readlane(tiles - more - 1 - place, which);
  tile_row = (uint32_t)tile * kTileRows;
}

template <typename E, int kQk, int kV, typename C>
__global__ __launch_bounds__(C::kThreads, kV == 64 && C::kWaves > 1 ? 3 : 1) void prompt_fwd(
    const int32_t* __restrict__ cu_q, const int32_t* __restrict__ cu_k, int32_t sequences, int32_t q_tokens,
    int32_t k_tokens, int32_t slots, int32_t splits, int32_t kv_heads, int32_t group_, const PromptArgs a) {
  constexpr int kWaves = C::kWaves, kTileRows = C::kRows;
  constexpr int kQuadsK = kQk / 32, kQuadsV = kV / 32;  // 64-byte column blocks
  constexpr int kStageK = kStageKeys * kQk * 2, kStageV = kStageKeys * kV * 2;
  constexpr int kSteps = kQk / 16, kDims = kV / 32;
  __shared__ __align__(1024) uint8_t lds[C::kBufK * kStageK + C::kBufV * kStageV];
  const uint32_t lds_k = (uint32_t)(uintptr_t)&lds[0], end_k = lds_k + C::kBufK * kStageK;
  const uint32_t lds_v = end_k, end_v = lds_v + C::kBufV * kStageV;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int n = lane & 31, h = lane >> 5;

  // ---- which row tile, KV head and split. Work-groups go round the XCDs by
  // linear id: with a multiple of 8 KV heads each XCD takes whole heads, whose
  // keys its L2 then holds. `rank` goes over the row tiles, longest first.
  // (All of this in 32 bits, which hold the rows of a call: with divisions of 64
  // bits and sequences found by bisection the start of a work-group took 5.3k cycles,
  // so 2.8k.)
  const uint32_t group = group_;
  const uint32_t unit = splits == 1 ? blockIdx.x : blockIdx.x / (uint32_t)splits;
  const int split = (int)(blockIdx.x - unit * (uint32_t)splits);
  int rank, kv_head;
  if (splits == 1 && kv_heads % 8 == 0) {
    const uint32_t in_xcd = unit >> 3, per_xcd = (uint32_t)kv_heads >> 3;
    rank = (int)(in_xcd / per_xcd);
    kv_head = (int)(in_xcd - rank * per_xcd) * 8 + (int)(unit & 7);
  } else {
    rank = (int)(unit / (uint32_t)kv_heads);
    kv_head = (int)(unit - rank * (uint32_t)kv_heads);
  }
  // Lane b looks at sequence lo + b of the up to 64 that the tile may be of; starts
  // outside the tensors are cut to them. Sequence b's tiles start at slot
  // cu_q[b] G / tile + b, which leaves room for a part-filled tile of every sequence
  // before it: a closed form, so a work-group finds its sequence with no plan made
  // beforehand. Later slots first: within a sequence later tiles see the most keys.
  const int slot = slots - 1 - rank;
  auto cut = [](int start, int tokens) -> int { return min(max(start, 0), tokens); };
  auto first_slot = [&](int start, int b) -> int { return (int)((uint32_t)start * group / kTileRows) + b; };
  int lo = 0;
  while (sequences > 64) {
    const int half = sequences >> 1;
    if (first_slot(cut(cu_q[lo + half], q_tokens), lo + half) <= slot) {
      lo += half;
      sequences -= half;
    } else {
      sequences = half;
    }
  }
  const int b = lo + min(lane, sequences - 1);
  const int lane_q = cut(cu_q[b], q_tokens), lane_k = cut(cu_k[b], k_tokens);
  const int lane_nq = max(cut(cu_q[b + 1], q_tokens) - lane_q, 0);
  const int lane_nk = max(cut(cu_k[b + 1], k_tokens) - lane_k, 0);
  int which;
  uint32_t tile_row = 0;
  if (kWaves > 1 && a.ranked) {
    const bool one = lane < sequences;
    tile_of_rank<kTileRows>(rank, group, a.causal, one ? lane_nq : 0, one ? lane_nk : 0, which, tile_row);
    if (which < 0) return;
  } else {
    // The last sequence whose first slot is <= slot.
    const int first = first_slot(lane_q, b);
    which = __builtin_popcountll(__builtin_amdgcn_ballot_w64(lane < sequences && first <= slot)) - 1;
    if (which < 0) return;
    tile_row = (uint32_t)(slot - __builtin_amdgcn_readlane(first, which)) * kTileRows;
  }
  const int64_t q_begin = __builtin_amdgcn_readlane(lane_q, which), k_begin = __builtin_amdgcn_readlane(lane_k, which);
  const int n_q = __builtin_amdgcn_readlane(lane_nq, which), n_k = __builtin_amdgcn_readlane(lane_nk, which);
  const uint32_t rows = (uint32_t)n_q * group;
  if (tile_row >= rows) return;

  // Keys that token i sees.
  auto visible = [&](uint32_t token) -> int {
    return a.causal ? max((int)token + 1 - n_q + n_k, 0) : n_k;
  };
  const uint32_t last_row = min(tile_row + kTileRows, rows) - 1;
  const int all_stages = (visible(last_row / group) + kStageKeys - 1) / kStageKeys;
  const int s0 = splits > 1 ? min(split * a.split_stages, all_stages) : 0;
  const int s1 = splits > 1 ? (split + 1 < splits ? min(s0 + a.split_stages, all_stages) : all_stages) : all_stages;

  // ---- this wave's 32 rows; lanes n and 32 + n have row n.
  const uint32_t wave_row = tile_row + wave * 32;
  const int wave_rows = wave_row < rows ? (int)min(32u, rows - wave_row) : 0;
  // Rows past the end repeat the last row; nothing of them is stored.
  const uint32_t r = min(wave_row + (uint32_t)n, rows - 1);
  const uint32_t token = r / group;
  const int head = (int)(kv_head * group + (r - token * group));
  const int sees = visible(token);
  // The stages this wave takes part in, and the first key that needs a mask.
  int w1 = s0, clear = 0;
  if (wave_rows > 0) {
    w1 = min(s1, (visible((wave_row + wave_rows - 1) / group) + kStageKeys - 1) / kStageKeys);
    clear = visible(wave_row / group);
  }
  w1 = __builtin_amdgcn_readfirstlane(w1);
  clear = __builtin_amdgcn_readfirstlane(clear);

  v4u q_ops[kSteps];
  {
    const uint16_t* src = a.q + (q_begin + token) * a.q_token + head * a.q_head + 8 * h;
#pragma unroll
    for (int ks = 0; ks < kSteps; ++ks) q_ops[ks] = *reinterpret_cast<const v4u*>(src + 16 * ks);
  }

  // ---- staging. A stage is two blocks of 16 rows by 64 bytes per column block,
  // dealt to the waves: four have one row block each and every other column block,
  // one has all.
  constexpr int kSpread = kWaves == 1 ? 2 : 1;  // row blocks of a wave
  constexpr int kLoadsK = 2 * kQuadsK / kWaves, kLoadsV = 2 * kQuadsV / kWaves, kLoads = kLoadsK + kLoadsV;
  static_assert(2 * kQuadsK % kWaves == 0 && 2 * kQuadsV % kWaves == 0, "blocks per wave");
  const uint8_t* k_from = reinterpret_cast<const uint8_t*>(a.k + (k_begin + (int64_t)s0 * kStageKeys) * a.k_token + kv_head * a.k_head);
  const uint8_t* v_from = reinterpret_cast<const uint8_t*>(a.v + (k_begin + (int64_t)s0 * kStageKeys) * a.v_token + kv_head * a.v_head);
  const int64_t k_stage = kStageKeys * a.k_token * 2, v_stage = kStageKeys * a.v_token * 2;
  const int load_row = 16 * (wave & 1) + (lane >> 2);
  const uint32_t load_at = 16u * ((lane & 3) ^ (lane >> 4)) + 64u * (wave >> 1);
  uint32_t k_off[kSpread], v_off[kSpread];
#pragma unroll
  for (int i = 0; i < kSpread; ++i) {
    k_off[i] = (uint32_t)(load_row + 16 * i) * (uint32_t)(a.k_token * 2) + load_at;
    v_off[i] = (uint32_t)(load_row + 16 * i) * (uint32_t)(a.v_token * 2) + load_at;
  }
  int to_load = s0;
  uint32_t k_to = lds_k, v_to = lds_v;
  auto issue = [&]() __attribute__((always_inline)) {
    if (to_load >= s1) return;
    if ((to_load + 1) * kStageKeys > n_k) {
      // Rows past the sequence's end repeat its last one: their scores are
      // masked, and what multiplies their zero probabilities is a row's own.
#pragma unroll
      for (int i = 0; i < kSpread; ++i) {
        const uint32_t row = (uint32_t)min(load_row + 16 * i, n_k - 1 - to_load * kStageKeys);
        k_off[i] = row * (uint32_t)(a.k_token * 2) + load_at;
        v_off[i] = row * (uint32_t)(a.v_token * 2) + load_at;
      }
    }
    // Column block c of a wave's i-th load; its place is 2048 bytes a column block
    // and 1024 a row block on. (A wave of four has c = 2 i + wave / 2.)
    static_for<kLoadsK>([&](auto i) {
      constexpr int c = kWaves == 1 ? i / 2 : 2 * i;
      load_to_lds<64 * c, 2048 * c + (kWaves == 1 ? 1024 * (i % 2) : 0)>(k_from, k_off[kWaves == 1 ? i % 2 : 0], k_to + 1024 * wave);
    });
    static_for<kLoadsV>([&](auto i) {
      constexpr int c = kWaves == 1 ? i / 2 : 2 * i;
      load_to_lds<64 * c, 2048 * c + (kWaves == 1 ? 1024 * (i % 2) : 0)>(v_from, v_off[kWaves == 1 ? i % 2 : 0], v_to + 1024 * wave);
    });
    ++to_load;
    k_from += k_stage;
    v_from += v_stage;
    k_to = k_to + kStageK == end_k ? lds_k : k_to + kStageK;
    v_to = v_to + kStageV == end_v ? lds_v : v_to + kStageV;
  };

  // LDS address of a stage's operands. K: key n, chunk 2 ks + h of its row; odd ks
  // flip chunk bit 1 (32 bytes). V: keys 16 t + 8 u + 4 h + jj, dims 32 d + 16 (g & 1)
  // + 4 qq; u flips chunk bit 1 and is 8 rows (512 bytes) on.
  const uint32_t k_lane = (uint32_t)(n >> 4) * 1024 + 64 * (n & 15) + 16 * (h ^ ((n & 15) >> 2));
  const uint32_t v_lane = (uint32_t)(64 * (4 * h + ((lane & 15) >> 2)) +
                                     16 * ((2 * ((lane >> 4) & 1) + ((lane & 3) >> 1)) ^ h) + 8 * (lane & 1));

  v16f o[kDims];
  RowState row{-__builtin_inff(), 0.0f};
  float shift = 0.0f;
#pragma unroll
  for (int d = 0; d < kDims; ++d) o[d] = v16f{};

  // Operands are read kAhead products ahead (in 64 dims, where three waves share
  // a SIMD, two).
  constexpr int kAhead = kV == 64 ? 2 : 4;
  constexpr int kVops = 2 * kDims;
  v4u kop[kAhead], vop[kAhead];
  auto read_k = [&](uint32_t at, int ks) __attribute__((always_inline)) {
    kop[ks % kAhead] = lds_load<v4u>((ks & 1 ? at ^ 32 : at) + 2048 * (ks >> 1));
  };
  auto read_v = [&](uint32_t at, int i) __attribute__((always_inline)) {
    const int t = i / kDims, d = i % kDims;
    const v2u lo = lds_column(at + 1024 * t + 2048 * d);
    const v2u hi = lds_column((at ^ 32) + 512 + 1024 * t + 2048 * d);
    vop[i % kAhead] = v4u{lo.x, lo.y, hi.x, hi.y};
  };
  // S of a stage (its first kAhead operands are in kop); `slice(i)` is issued
  // after product i: independent work that the matrix unit leaves room for.
  auto scores = [&](uint32_t at, v16f& s, auto slice) __attribute__((always_inline)) {
    s = v16f{};
#pragma unroll
    for (int ks = 0; ks < kSteps; ++ks) {
      s = E::mfma(kop[ks % kAhead], q_ops[ks], s);
      if (ks + kAhead < kSteps) read_k(at, ks + kAhead);
      slice(ks);
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  // O^T += V^T P^T of a stage (its first kAhead operands are in vop).
  auto values = [&](uint32_t at, const v4u (&p)[2], auto slice) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < kVops; ++i) {
      o[i % kDims] = E::mfma(vop[i % kAhead], p[i / kDims], o[i % kDims]);
      if (i + kAhead < kVops) read_v(at, i + kAhead);
      slice(i);
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  // Keys a row does not see: -inf.
  auto mask = [&](int j, v16f& s) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < 16; ++i)
      s[i] = kStageKeys * j + 8 * (i >> 2) + 4 * h + (i & 3) < sees ? s[i] : -__builtin_inff();
  };
  // The next stage has landed for this wave (those after it may be in flight), then
  // for every wave, which are then also done with the K of the stage before and the
  // V of the two before that.
  int entered = s0;  // stages entered so far end here
  auto enter_stage = [&]() __attribute__((always_inline)) {
    if (entered + C::kDistance <= s1) wait_loads<(C::kDistance - 1) * kLoads>(); else wait_loads<0>();
    lds_barrier();
    issue();
    ++entered;
  };
  static_assert((C::kDistance - 1) * kLoads < 64, "outstanding loads");

#pragma unroll
  for (int i = 0; i < C::kDistance; ++i) issue();
  if (w1 > s0) {
    int j = s0;
    uint32_t k_ring = lds_k, v_ring = lds_v;                // of stage j
    uint32_t k_at = lds_k + k_lane, v_at = lds_v + v_lane;  // and this lane's place there
    auto next_k = [&]() {
      k_ring = __builtin_amdgcn_readfirstlane(k_ring + kStageK == end_k ? lds_k : k_ring + kStageK);
      k_at = opaque(k_ring + k_lane);
    };
    auto next_v = [&]() {
      v_ring = __builtin_amdgcn_readfirstlane(v_ring + kStageV == end_v ? lds_v : v_ring + kStageV);
      v_at = opaque(v_ring + v_lane);
    };
    v16f s, next;
    v4u p[2];
    constexpr int kPairs = 8, kTicks = kPairs + 2;
    auto no_slice = [](int) {};
    Softener<E> softener;
    // Slice i of `of` of the probabilities of the scores in `from`.
    auto soften = [&](const v16f& from, int i, int of) __attribute__((always_inline)) {
#pragma unroll
      for (int u = kTicks * i / of; u < kTicks * (i + 1) / of; ++u)
        softener.tick(u, kPairs, a.scale_log2, [&](int e) { return from[e]; }, &shift, [&](int w, uint32_t pair) {
          p[w >> 2][w & 3] = pair;
          row.sum = E::add_pair(pair, row.sum);
        });
    };
    // One step: stage j's scores beside the probabilities of stage j - 1 (scores in
    // `from`, its rows' maxima raised), then stage j - 1's product with V beside the
    // maxima of stage j (into `to`) and the first K reads of stage j + 1, which is
    // entered between the two. Says whether the inner loop ends: a row's maximum
    // must rise or the stage needs a mask (kBreak), or there was no stage left
    // (kDone, `to` not written).
    enum { kGo, kBreak, kDone };
    auto step = [&](const v16f& from, v16f& to) __attribute__((always_inline)) -> int {
      if (j + 1 == w1) return kDone;
      ++j;
      scores(k_at, to, [&](int i) __attribute__((always_inline)) {
        soften(from, i, kSteps);
#pragma unroll
        for (int u = 0; u < kAhead; ++u)
          if (i == kSteps - 1 - kAhead + u || (kSteps < kAhead + 1 && i == kSteps - 1)) read_v(v_at, u);
      });
      // Computed by here, beside the products, not where they are used.
      asm volatile("" : "+v"(p[0]), "+v"(p[1]), "+v"(row.sum));
      if (j + 1 < s1) enter_stage();
      next_k();
      float top = -__builtin_inff();
      uint64_t rise = 0;
      values(v_at, p, [&](int i) __attribute__((always_inline)) {
        // Pairs of scores over half of the products, the check, the reads.
        constexpr int kPerSlot = kVops >= 8 ? 2 : 4;
#pragma unroll
        for (int u = kPerSlot * i; u < kPerSlot * (i + 1) && u < kPairs; ++u)
          top = fmaxf(fmaxf(top, to[2 * u]), to[2 * u + 1]);
        if (i == kPairs / kPerSlot)
          rise = __builtin_amdgcn_ballot_w64(must_raise<E>(row, max_halves(top) * a.scale_log2));
        if (i >= kVops - kAhead) read_k(k_at, i - (kVops - kAhead));
      });
      next_v();
      return kStageKeys * (j + 1) > clear || rise != 0 ? kBreak : kGo;
    };
    enter_stage();
#pragma unroll
    for (int ks = 0; ks < kAhead; ++ks) read_k(k_at, ks);
    scores(k_at, s, no_slice);
    if (s0 + 1 < s1) enter_stage();
    next_k();
#pragma unroll
    for (int ks = 0; ks < kAhead; ++ks) read_k(k_at, ks);
    // Masks, and the rise of a row's maximum (by which what it summed so far is
    // rescaled), stay outside the inner loop: a multiply of the accumulators in
    // it makes the compiler keep a second copy of them and spill.
    for (bool more = true; more;) {
      if (kStageKeys * (j + 1) > clear) mask(j, s);
      const float factor = raise<E>(row, row_max(s, a.scale_log2));
      shift = shift_of(row);
      if (__builtin_amdgcn_ballot_w64(factor != 1.0f)) {
#pragma unroll
        for (int d = 0; d < kDims; ++d) o[d] *= factor;
      }
      for (;;) {
        int end = step(s, next);
        if (end != kGo) {
          more = end == kBreak;
          if (more) s = next;
          break;
        }
        end = step(next, s);
        if (end != kGo) {
          more = end == kBreak;
          if (!more) s = next;
          break;
        }
      }
    }
#pragma unroll
    for (int i = 0; i < kAhead; ++i) read_v(v_at, i);
    soften(s, 0, 1);
    values(v_at, p, no_slice);
  }
  while (entered < s1) enter_stage();

  // ---- store. A lane holds dims 32 d + 8 b + 4 h + 0 .. 3 of its row; the halves
  // trade so that each stores 16 bytes.
  const float sum = sum_halves(row.sum);
  const bool live = n < wave_rows;
  const int64_t at = (q_begin + token) * a.heads + head;
  if (splits > 1) {
    const int64_t part = (int64_t)split * q_tokens * a.heads + at;
    if (live && h == 0) a.stats[part] = split_stats(row.top, sum);
    if (live && sum != 0.0f) {
#pragma unroll
      for (int d = 0; d < kDims; ++d)
#pragma unroll
        for (int b = 0; b < 4; ++b)
          *reinterpret_cast<v4f*>(a.parts + part * kV + 32 * d + 8 * b + 4 * h) =
              v4f{o[d][4 * b], o[d][4 * b + 1], o[d][4 * b + 2], o[d][4 * b + 3]};
    }
    return;
  }
  const float inv = sum > 0.0f ? 1.0f / sum : (sum == 0.0f ? 0.0f : sum);
#pragma unroll
  for (int d = 0; d < kDims; ++d)
#pragma unroll
    for (int b = 0; b < 4; b += 2) {
      uint32_t w[2][2];
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int e = 0; e < 2; ++e)
          w[u][e] = E::pack(o[d][4 * (b + u) + 2 * e] * inv, o[d][4 * (b + u) + 2 * e + 1] * inv);
      const auto x = __builtin_amdgcn_permlane32_swap(w[0][0], w[1][0], false, false);
      const auto y = __builtin_amdgcn_permlane32_swap(w[0][1], w[1][1], false, false);
      if (live) *reinterpret_cast<v4u*>(a.out + at * kV + 32 * d + 8 * (b + h)) = v4u{x[0], y[0], x[1], y[1]};
    }
}

// The cut of a call. Rows of a sequence and KV head that fill a wave at most (single
// tokens): work-groups of one wave, two of them per CU; a wave alone in a work-group
// of several would walk every key by itself, which bounds the call, not memory (8 single
// tokens over 40,000 keys 67 -> 44 us). Others: four waves, 128 rows.
using FewRows = Cut<1, 2>;
using ManyRows = Cut<4, 2>;

// Key splits, where the row tiles are too few for the chip: ranges of the same
// number of stages, so that sequences of different lengths make work-groups of the
// same size.
// The count of least time (split_us), fitted to 11 calls of 1 to 24 single tokens over
// 500 to 60,000 keys and 12 of 64 to 3,000 queries over up to 65,600, each with 1 to 48
// splits.
constexpr int64_t kMinSplitStages = 8, kMaxSplits = 256;

struct PromptPlan {
  bool few, ranked;
  int64_t slots, splits, split_stages, bytes, stats_at;
};

// Time of a call whose keys are split into ranges of `of` of at most `stages` stages
// (about `seen` on average): a work-group takes 0.62 us a stage alone on its CU and, if
// it has four waves, 1.15 where the CU has two, and 5 us beside them; reading K and V once
// bounds all of them (`apart`: adds to their own time, as the root of the sum of both
// squared: with few loads on their way neither hides the other); the parts of each row
// are written and read again.
double split_us(bool few, bool apart, double tiles, double seen, double stages, double of, double rows, double v_dim,
                double kv_bytes, double cus) {
  const double scale = 0.5 + v_dim / 256, fixed = 5.0, alone = 0.62 * scale, shared = 1.15 * scale;
  const double parts = of < stages ? __builtin_ceil((seen + stages) / 2 / of) : 1.0;
  const double groups = tiles * parts, total = tiles * seen;
  double us = fixed + alone * of;
  if (few) {
    us *= __builtin_ceil(groups / (2 * cus));
  } else if (groups > 2 * cus) {
    us = (total * shared + groups * fixed) / (2 * cus) + 0.25 * (fixed + shared * of);
  } else if (groups > cus) {
    const double load = total / (2 * cus * of);
    us += (shared - alone) * (load < 1.0 ? load : 1.0) * of;
  }
  const double read = kv_bytes / 5.5e6;
  us = apart ? __builtin_sqrt(us * us + read * read) : us < read ? read : us;
  return of < stages ? us + 4.0 + rows * parts * v_dim * 8 / 3.4e6 : us;
}

PromptPlan prompt_plan(int64_t q_tokens, int64_t heads, int64_t kv_heads, int64_t v_dim, int64_t sequences,
                       int64_t k_tokens, int64_t max_k) {
  PromptPlan p{};
  // (Stages of no more than k_tokens keys stay within the kernel's 32 bits.)
  if (max_k > k_tokens) max_k = k_tokens;
  const int64_t rows = q_tokens * (heads / kv_heads);
  p.few = rows <= FewRows::kRows * sequences;
  p.slots = rows / (p.few ? FewRows::kRows : ManyRows::kRows) + sequences;
  const int64_t units = p.slots * kv_heads;
  const int64_t round = 2 * device_cu_count();  // two work-groups per CU
  // Tiles by rank where the work-groups are at most two rounds: 4,434 tokens in 8
  // sequences, 16 heads of 192 / 128 (672 work-groups) 34.7 -> 31.5 us, 3,000 in 3, 32
  // heads of 128 (832) 46.9 -> 45.2. With more, neighbours of different sequences cost
  // more in L2 than the order gives: 32 heads of the first (1,344) 52.7 -> 58.7.
  p.ranked = !p.few && sequences > 1 && sequences <= 64 && units <= 2 * round;
  p.splits = 1;
  // Stages of a row tile, if a sequence is as long as the others, and of the longest
  // (taken for twice that, of single tokens four times, where it is not given).
  const int64_t mean = k_tokens / kStageKeys / sequences + 1;
  int64_t stages = ((max_k < 0 ? k_tokens : max_k) + kStageKeys - 1) / kStageKeys;
  if (max_k < 0 && stages > (p.few ? 4 : 2) * mean) stages = (p.few ? 4 : 2) * mean;
  if (units < round && stages > kMinSplitStages) {
    const int64_t tile = p.few ? FewRows::kRows : ManyRows::kRows;
    const double tiles = (double)(sequences * kv_heads) * (double)((rows + tile * sequences - 1) / (tile * sequences));
    double seen = ((double)k_tokens - 0.5 * (double)q_tokens) / (double)(sequences * kStageKeys);
    if (seen > (double)stages) seen = (double)stages;
    if (seen < 1.0) seen = 1.0;
    const double kv_bytes = 4.5 * (double)(k_tokens * kv_heads * v_dim);  // (its two dims together are about 2.25)
    const auto us = [&](int64_t of, bool apart) {
      return split_us(p.few, apart, tiles, seen, (double)stages, (double)of, (double)(rows * kv_heads), (double)v_dim,
                      kv_bytes, (double)(round / 2));
    };
    p.split_stages = stages;
    double least = us(stages, false);
    for (int64_t s = 2; s <= kMaxSplits; s += s < 8 ? 1 : s < 16 ? 2 : s < 32 ? 4 : s < 64 ? 8 : 32) {
      const int64_t of = (stages + s - 1) / s;
      if (of < kMinSplitStages) break;
      if (const double t = us(of, false); t < least) {
        least = t;
        p.split_stages = of;
      }
    }
    // Single tokens: or two rounds of work-groups, which keep more loads on their way (4
    // over 30,000 keys, 16 heads of 192 / 128: 63 us, with five splits 78).
    if (p.few) {
      int64_t of = (units * (mean < stages ? mean : stages) + 2 * round - 1) / (2 * round);
      if (of < kMinSplitStages) of = kMinSplitStages;
      if (us(of, true) < us(p.split_stages, true)) p.split_stages = of;
    }
    if (p.split_stages < (stages + kMaxSplits - 1) / kMaxSplits) p.split_stages = (stages + kMaxSplits - 1) / kMaxSplits;
    if (p.split_stages < kMinSplitStages) p.split_stages = kMinSplitStages;
    p.splits = (stages + p.split_stages - 1) / p.split_stages;
  }
  if (p.splits > 1) {
    p.stats_at = p.splits * q_tokens * heads * v_dim * 4;
    p.bytes = p.stats_at + p.splits * q_tokens * heads * 8;
  }
  return p;
}

struct PromptCall {
  const int32_t *cu_q, *cu_k;
  int64_t sequences, q_tokens, k_tokens, kv_heads;
  PromptPlan plan;
  PromptArgs args;
};

template <typename E, int kQk, int kV>
int launch_prompt(const PromptCall& c, hipStream_t stream) {
  const auto go = [&](auto kernel, int threads) {
    hipLaunchKernelGGL(kernel, dim3((unsigned)(c.plan.slots * c.kv_heads * c.plan.splits)), dim3(threads), 0, stream,
                       c.cu_q, c.cu_k, (int32_t)c.sequences, (int32_t)c.q_tokens, (int32_t)c.k_tokens,
                       (int32_t)c.plan.slots, (int32_t)c.plan.splits, (int32_t)c.kv_heads,
                       (int32_t)(c.args.heads / c.kv_heads), c.args);
  };
  if (c.plan.few) go(prompt_fwd<E, kQk, kV, FewRows>, FewRows::kThreads);
  else go(prompt_fwd<E, kQk, kV, ManyRows>, ManyRows::kThreads);
  DSA_CHECK_LAUNCH("prompt attention");
  if (c.plan.splits > 1)
    return launch_join<E, kV>(c.args.parts, c.args.stats, c.q_tokens * c.args.heads, (int)c.plan.splits, c.cu_q,
                              (int32_t)c.sequences, c.args.heads, c.args.out, stream);
  return kOk;
}

template <typename E>
int launch_dims(const PromptCall& c, int64_t qk_dim, int64_t v_dim, hipStream_t stream) {
  if (qk_dim == 192 && v_dim == 128) return launch_prompt<E, 192, 128>(c, stream);
  if (qk_dim == 128 && v_dim == 128) return launch_prompt<E, 128, 128>(c, stream);
  return launch_prompt<E, 64, 64>(c, stream);
}

// What the plan's and the kernel's arithmetic is made for.
int check_sizes(int64_t q_tokens, int64_t heads, int64_t kv_heads, int64_t sequences, int64_t k_tokens) {
  DSA_CHECK_ARG(heads > 0 && kv_heads > 0 && heads % kv_heads == 0 && heads <= 65536,
                "heads must be a positive multiple of kv_heads");
  // (Rounding up to a stage must stay within int32.)
  constexpr int64_t kMost = 0x7FFFFFFF - kStageKeys;
  DSA_CHECK_ARG(q_tokens >= 0 && k_tokens >= 0 && q_tokens <= kMost && k_tokens <= kMost && sequences >= 0 &&
                    sequences <= kMost,
                "token and sequence counts must be in [0, 2^31 - 33]");
  DSA_CHECK_ARG(q_tokens * heads < 0x7FFFFF00, "too many query rows");
  return kOk;
}

}  // namespace
}  // namespace dsa

extern "C" int dsa_prompt_attention_workspace_bytes(int64_t q_tokens, int64_t heads, int64_t kv_heads, int64_t v_dim,
                                                    int64_t sequences, int64_t k_tokens, int64_t max_k, int64_t* bytes) {
  using namespace dsa;
  DSA_CHECK_ARG(bytes != nullptr, "null pointer");
  DSA_CHECK_ARG(q_tokens >= 0 && sequences >= 0 && k_tokens >= 0 && v_dim > 0 && v_dim <= 128,
                "invalid prompt attention shape");
  if (const int status = check_sizes(q_tokens, heads, kv_heads, sequences, k_tokens); status != kOk) return status;
  *bytes = sequences == 0 ? 0 : prompt_plan(q_tokens, heads, kv_heads, v_dim, sequences, k_tokens, max_k).bytes;
  return kOk;
}

extern "C" int dsa_prompt_attention(const void* q, int64_t q_token_stride, int64_t q_head_stride, const void* k,
                                    int64_t k_token_stride, int64_t k_head_stride, const void* v,
                                    int64_t v_token_stride, int64_t v_head_stride, int dtype, int64_t heads,
                                    int64_t kv_heads, int64_t qk_dim, int64_t v_dim, const int32_t* cu_q,
                                    const int32_t* cu_k, int64_t sequences, int64_t q_tokens, int64_t k_tokens,
                                    int64_t max_k, float scale, int causal, void* out, void* workspace,
                                    int64_t workspace_bytes, hipStream_t stream) {
  using namespace dsa;
  DSA_CHECK_ARG(dtype == DSA_DTYPE_BF16 || dtype == DSA_DTYPE_F16, "prompt attention takes bf16 or fp16");
  DSA_CHECK_ARG((qk_dim == 192 && v_dim == 128) || (qk_dim == 128 && v_dim == 128) || (qk_dim == 64 && v_dim == 64),
                "head dims must be (192, 128), (128, 128) or (64, 64)");
  if (const int status = check_sizes(q_tokens, heads, kv_heads, sequences, k_tokens); status != kOk) return status;
  DSA_CHECK_ARG(scale > 0.0f && __builtin_isfinite(scale), "scale must be positive and finite");
  if (q_tokens == 0) return kOk;
  DSA_CHECK_ARG(sequences > 0, "queries need a sequence");
  DSA_CHECK_ARG(q && out && cu_q && cu_k && (k_tokens == 0 || (k && v)), "null pointer");
  const int64_t strides[] = {q_token_stride, q_head_stride, k_token_stride, k_head_stride, v_token_stride, v_head_stride};
  for (int64_t s : strides)
    DSA_CHECK_ARG(s % 8 == 0 && s >= 0 && s < (1ll << 25), "strides must be multiples of 8 elements below 2^25");
  DSA_CHECK_ARG((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v) |
                 reinterpret_cast<uintptr_t>(out)) % 16 == 0,
                "q, k, v and out must be 16-byte aligned");
  const PromptPlan p = prompt_plan(q_tokens, heads, kv_heads, v_dim, sequences, k_tokens, max_k);
  // (A call with splits has less than two rounds of row tiles, so its join is small.)
  DSA_CHECK_ARG(p.slots <= 0xFFFFFFFFll / kv_heads / p.splits &&
                    grid_fits(p.slots * kv_heads * p.splits, p.few ? FewRows::kThreads : ManyRows::kThreads),
                "too many query rows or sequences");
  if (p.splits > 1)
    DSA_CHECK_ARG(workspace && reinterpret_cast<uintptr_t>(workspace) % 16 == 0 && workspace_bytes >= p.bytes,
                  "prompt attention workspace too small or misaligned");
  PromptCall c{cu_q, cu_k, sequences, q_tokens, k_tokens, kv_heads, p, {}};
  PromptArgs& a = c.args;
  a.q = static_cast<const uint16_t*>(q);
  a.k = static_cast<const uint16_t*>(k);
  a.v = static_cast<const uint16_t*>(v);
  a.out = static_cast<uint16_t*>(out);
  a.parts = static_cast<float*>(workspace);
  a.stats = reinterpret_cast<float2*>(static_cast<uint8_t*>(workspace) + p.stats_at);
  a.q_token = q_token_stride, a.q_head = q_head_stride;
  a.k_token = k_token_stride, a.k_head = k_head_stride;
  a.v_token = v_token_stride, a.v_head = v_head_stride;
  a.heads = (int32_t)heads, a.split_stages = (int32_t)p.split_stages;
  a.causal = causal != 0, a.ranked = p.ranked;
  a.scale_log2 = scale * kLog2E;
  return dtype == DSA_DTYPE_BF16 ? launch_dims<Bf16>(c, qk_dim, v_dim, stream)
                                 : launch_dims<F16>(c, qk_dim, v_dim, stream);
}
