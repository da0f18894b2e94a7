// Causal attention over packed sequences with grouped heads, forward.
//
// Per sequence of n_q queries and n_k keys, head h of H reading KV head
// h / G (G = H / H_kv): out = softmax(scale q k^T) v over the keys
// j <= i + n_k - n_q of query i (causal; every key otherwise), in fp32 from
// 16-bit inputs, probabilities rounded to 16 bits before the product with V;
// a query without a visible key gives zeros. 2 (d_qk + d_v) flop per pair.
//
// Mapping (gfx950, wave64). The G heads that share a KV head are rows of one
// problem: row r of a sequence is token r / G, head r % G, so that single tokens
// of grouped heads fill a tile and K and V are staged once for all of them. A
// work-group of four waves (one per SIMD) owns 256 rows, 64 per wave, and walks
// the keys in stages of 64. A wave computes S^T = K Q^T (v_mfma_f32_32x32x16,
// Q^T in registers) for 32 keys at a time and its two tiles of 32 rows: each
// operand read from LDS feeds two products, which keeps LDS at half of what it
// can deliver (64 of ~115 B a cycle with one wave per SIMD; with 32 rows per
// wave it would be the bound). The result's layout - a lane holds 16 keys of one
// row - is the operand layout of O^T += V^T P^T once the keys of V^T are read in
// the same order, so probabilities never leave registers and a row's softmax
// state and rescale factor belong to its lane.
// Software pipeline: the products S of 32 keys run beside the softmax of the 32
// keys before, then those keys' product with V.
//
// Stages arrive by LDS DMA two ahead, in blocks of 16 rows by 64 bytes: lane l
// brings chunk (l % 4) ^ (l / 16) (16 bytes) of row l / 4, which makes global
// reads whole 64-byte segments and both the K reads (16 rows, one chunk) and the
// transposing V reads (4 rows, 4 chunks) free of bank conflicts.
#include "attention_core.h"
#include "../../include/dsa_gfx950.h"

namespace dsa {
namespace {

constexpr int kThreads = 256;
constexpr int kWaveRows = 64;
constexpr int kTileRows = 4 * kWaveRows;
constexpr int kStageKeys = 64;

struct PromptArgs {
  const uint16_t* q;
  const uint16_t* k;
  const uint16_t* v;
  const int32_t* cu_q;
  const int32_t* cu_k;
  uint16_t* out;
  float* parts;    // [splits][q_tokens * heads][d_v], splits > 1 only
  float2* stats;   // [splits][q_tokens * heads]
  int64_t q_token, q_head, k_token, k_head, v_token, v_head;  // strides, elements
  int64_t q_tokens, k_tokens;
  int32_t heads, kv_heads, sequences, slots, splits, causal;
  float scale_log2;
};

// Slots of row tiles: sequence b's tiles start at slot cu_q[b] G / 256 + b, which
// leaves room for a part-filled tile of every sequence before it: a closed form,
// so a work-group finds its sequence by bisection, with no plan made beforehand.
__host__ __device__ inline int64_t first_slot(int64_t start, int64_t group, int64_t b) {
  return start * group / kTileRows + b;
}

template <typename E, int kQk, int kV>
__global__ __launch_bounds__(kThreads, 1) void prompt_fwd(const PromptArgs a) {
  constexpr int kQuadsK = kQk / 32, kQuadsV = kV / 32;  // 64-byte column blocks
  constexpr int kStageK = kStageKeys * kQk * 2, kStageV = kStageKeys * kV * 2;
  constexpr int kBufK = 3, kBufV = 4;
  constexpr int kSteps = kQk / 16, kDims = kV / 32;
  __shared__ __align__(1024) uint8_t lds[kBufK * kStageK + kBufV * kStageV];
  const uint32_t lds_k = (uint32_t)(uintptr_t)&lds[0];
  const uint32_t lds_v = lds_k + kBufK * kStageK;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int n = lane & 31, h = lane >> 5;

  // ---- which row tile, KV head and split. Work-groups go round the XCDs by
  // linear id: with a multiple of 8 KV heads each XCD takes whole heads, whose
  // keys its L2 then holds. Later tiles first: under a causal mask they see the
  // most keys.
  const int group = a.heads / a.kv_heads;
  int64_t unit = blockIdx.x / a.splits;
  const int split = (int)(blockIdx.x % a.splits);
  int slot, kv_head;
  if (a.splits == 1 && a.kv_heads % 8 == 0) {
    const int64_t in_xcd = unit >> 3;
    kv_head = (int)(in_xcd / a.slots) * 8 + (int)(unit & 7);
    slot = a.slots - 1 - (int)(in_xcd % a.slots);
  } else {
    kv_head = (int)(unit % a.kv_heads);
    slot = a.slots - 1 - (int)(unit / a.kv_heads);
  }
  int lo = 0, hi = a.sequences;  // the last sequence whose first slot is <= slot
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (first_slot(a.cu_q[mid], group, mid) <= slot) lo = mid; else hi = mid;
  }
  // Lengths outside the tensors are cut to them.
  const int64_t q_begin = min(max((int64_t)a.cu_q[lo], (int64_t)0), a.q_tokens);
  const int64_t q_end = min(max((int64_t)a.cu_q[lo + 1], q_begin), a.q_tokens);
  const int64_t k_begin = min(max((int64_t)a.cu_k[lo], (int64_t)0), a.k_tokens);
  const int64_t k_end = min(max((int64_t)a.cu_k[lo + 1], k_begin), a.k_tokens);
  const int n_q = (int)(q_end - q_begin), n_k = (int)(k_end - k_begin);
  const int64_t tile_row = ((int64_t)slot - first_slot(a.cu_q[lo], group, lo)) * kTileRows;
  const int64_t rows = (int64_t)n_q * group;
  if (tile_row < 0 || tile_row >= rows) return;

  // Keys that token i sees.
  auto visible = [&](int64_t token) -> int {
    if (!a.causal) return n_k;
    const int64_t m = token + 1 + n_k - n_q;
    return (int)min(max(m, (int64_t)0), (int64_t)n_k);
  };
  const int64_t last_row = min(tile_row + kTileRows, rows) - 1;
  const int all_stages = (visible(last_row / group) + kStageKeys - 1) / kStageKeys;
  const int per_split = (all_stages + a.splits - 1) / a.splits;
  const int s0 = split * per_split;
  const int s1 = min(s0 + per_split, all_stages);

  // ---- this wave's rows: two tiles of 32, this lane's rows n and 32 + n.
  const int64_t wave_row = tile_row + wave * kWaveRows;
  const int wave_rows = (int)min((int64_t)kWaveRows, rows - wave_row);  // may be <= 0
  int64_t token[2];
  int head[2], sees[2];
#pragma unroll
  for (int t = 0; t < 2; ++t) {
    // Rows past the end repeat the wave's last row; nothing of them is stored.
    const int64_t row = wave_row + min(32 * t + n, max(wave_rows - 1, 0));
    const int64_t r = min(row, rows - 1);
    token[t] = r / group;
    head[t] = kv_head * group + (int)(r - token[t] * group);
    sees[t] = visible(token[t]);
  }
  // The stages this wave takes part in, and the first 32 keys that need a mask.
  int w1 = s0, clear = 0;
  if (wave_rows > 0) {
    w1 = min(s1, (visible((wave_row + wave_rows - 1) / group) + kStageKeys - 1) / kStageKeys);
    clear = visible(wave_row / group);
  }
  w1 = __builtin_amdgcn_readfirstlane(w1);
  clear = __builtin_amdgcn_readfirstlane(clear);

  v4u q_ops[2][kSteps];
#pragma unroll
  for (int t = 0; t < 2; ++t) {
    const uint16_t* src = a.q + (q_begin + token[t]) * a.q_token + head[t] * a.q_head + 8 * h;
#pragma unroll
    for (int ks = 0; ks < kSteps; ++ks) q_ops[t][ks] = *reinterpret_cast<const v4u*>(src + 16 * ks);
  }
  // In AGPRs, from where the products read their second operand: VGPRs are left
  // to the accumulators and the softmax.
#pragma unroll
  for (int t = 0; t < 2; ++t)
#pragma unroll
    for (int ks = 0; ks < kSteps; ++ks) asm volatile("" : "+a"(q_ops[t][ks]));

  // ---- staging. Wave w brings rows 16 w .. + 15 of every column block.
  const uint8_t* k_base = reinterpret_cast<const uint8_t*>(a.k + k_begin * a.k_token + kv_head * a.k_head);
  const uint8_t* v_base = reinterpret_cast<const uint8_t*>(a.v + k_begin * a.v_token + kv_head * a.v_head);
  const int load_row = 16 * wave + (lane >> 2);
  const uint32_t load_chunk = 16u * ((lane & 3) ^ (lane >> 4));
  auto issue = [&](int stage) {
    if (stage >= s1) return;
    // Rows past the sequence's end repeat its last one: their scores are
    // masked, and what multiplies their zero probabilities is a row's own.
    const int64_t key0 = (int64_t)stage * kStageKeys;
    const uint32_t row = (uint32_t)min((int64_t)load_row, n_k - 1 - key0);
    const uint8_t* kb = k_base + key0 * a.k_token * 2;
    const uint8_t* vb = v_base + key0 * a.v_token * 2;
    const uint32_t k_off = row * (uint32_t)(a.k_token * 2) + load_chunk;
    const uint32_t v_off = row * (uint32_t)(a.v_token * 2) + load_chunk;
    const uint32_t kl = lds_k + (uint32_t)(stage % kBufK) * kStageK + 1024 * wave;
    const uint32_t vl = lds_v + (uint32_t)(stage % kBufV) * kStageV + 1024 * wave;
#pragma unroll
    for (int c = 0; c < kQuadsK; ++c) load_to_lds(kb + 64 * c, k_off, kl + 4096 * c);
#pragma unroll
    for (int c = 0; c < kQuadsV; ++c) load_to_lds(vb + 64 * c, v_off, vl + 4096 * c);
  };
  constexpr int kLoads = kQuadsK + kQuadsV;

  // LDS address of a stage's operands. K: key 32 half + n, chunk 2 ks + h of its
  // row; odd ks flip chunk bit 1. V: keys 16 t + 8 u + 4 h + jj, dims
  // 32 d + 16 (g & 1) + 4 qq; u flips chunk bit 1.
  uint32_t k_lane[2], v_lane[2];
#pragma unroll
  for (int o = 0; o < 2; ++o) {
    k_lane[o] = (uint32_t)(n >> 4) * 1024 + 64 * (n & 15) + 16 * ((2 * o + h) ^ ((n & 15) >> 2));
    const int jj = (lane & 15) >> 2, qq = lane & 3, g1 = (lane >> 4) & 1;
    v_lane[o] = 64 * (8 * o + 4 * h + jj) + 16 * ((2 * g1 + (qq >> 1)) ^ (2 * o + h)) + 8 * (qq & 1);
  }

  v16f o[2][kDims];
#pragma unroll
  for (int t = 0; t < 2; ++t)
#pragma unroll
    for (int d = 0; d < kDims; ++d) o[t][d] = v16f{};
  RowState row[2] = {{-__builtin_inff(), 0.0f}, {-__builtin_inff(), 0.0f}};

  // Block j: keys 32 j .. + 31, half j % 2 of stage j / 2.
  auto k_at = [&](int j, int odd) -> uint32_t {
    return opaque_address(lds_k + (uint32_t)((j >> 1) % kBufK) * kStageK + 2048 * (j & 1) + k_lane[odd]);
  };
  auto v_at = [&](int j, int upper) -> uint32_t {
    return opaque_address(lds_v + (uint32_t)((j >> 1) % kBufV) * kStageV + 2048 * (j & 1) + v_lane[upper]);
  };
  constexpr int kAhead = 4;  // operands read ahead of their product
  constexpr int kVops = 2 * kDims;
  // S of block j (both row tiles); `slice(i)`, i < 2 kSteps, is issued after
  // product i: independent work that the matrix unit leaves room for.
  auto scores = [&](int j, v16f (&s)[2], auto slice) __attribute__((always_inline)) {
    const uint32_t at[2] = {k_at(j, 0), k_at(j, 1)};
    v4u kop[kAhead];
#pragma unroll
    for (int ks = 0; ks < kAhead; ++ks) kop[ks] = lds_load<v4u>(at[ks & 1] + 4096 * (ks >> 1));
    s[0] = v16f{};
    s[1] = v16f{};
#pragma unroll
    for (int ks = 0; ks < kSteps; ++ks) {
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        s[t] = E::mfma(kop[ks % kAhead], q_ops[t][ks], s[t]);
        if (t == 1 && ks + kAhead < kSteps)
          kop[ks % kAhead] = lds_load<v4u>(at[ks & 1] + 4096 * ((ks + kAhead) >> 1));
        slice(2 * ks + t);
        __builtin_amdgcn_sched_barrier(0);
      }
    }
  };
  auto read_v = [&](const uint32_t (&at)[2], int i) __attribute__((always_inline)) -> v4u {
    const int t = i / kDims, d = i % kDims;
    const v2u lo = lds_column(at[0] + 1024 * t + 4096 * d);
    const v2u hi = lds_column(at[1] + 1024 * t + 4096 * d);
    return v4u{lo.x, lo.y, hi.x, hi.y};
  };
  // O^T += V^T P^T of block j, whose first operands are in vop.
  auto values = [&](const uint32_t (&at)[2], v4u (&vop)[kAhead], const v4u (&p)[2][2], auto slice)
                    __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < kVops; ++i) {
      const int t = i / kDims, d = i % kDims;
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        o[r][d] = E::mfma(vop[i % kAhead], p[r][t], o[r][d]);
        if (r == 1 && i + kAhead < kVops) vop[i % kAhead] = read_v(at, i + kAhead);
        slice(2 * i + r);
        __builtin_amdgcn_sched_barrier(0);
      }
    }
  };
  // Keys a row does not see: -inf.
  auto mask = [&](int j, v16f (&s)[2]) __attribute__((always_inline)) {
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int i = 0; i < 16; ++i)
        s[t][i] = 32 * j + 8 * (i >> 2) + 4 * h + (i & 3) < sees[t] ? s[t][i] : -__builtin_inff();
  };
  // The stage has landed for this wave (the loads of the next may be in flight),
  // then for every wave, which are then also done with the stage before.
  auto enter_stage = [&](int stage) {
    if (stage + 1 < s1) wait_loads<kLoads>(); else wait_loads<0>();
    lds_barrier();
    issue(stage + 2);
  };

  issue(s0);
  issue(s0 + 1);
  if (w1 > s0) {
    const int j1 = 2 * w1;
    int j = 2 * s0;
    v16f s[2], next[2];
    v4u p[2][2];
    float shift[2];
    auto no_slice = [](int) {};
    // Slice i of n: the 16 pairs of probabilities of both rows.
    auto soften = [&](const v16f (&from)[2], int i, int n) __attribute__((always_inline)) {
#pragma unroll
      for (int u = 16 * i / n; u < 16 * (i + 1) / n; ++u) {
        const int t = u >> 3, w = u & 7;
        p[t][w >> 2][w & 3] =
            probability_pair<E>(from[t][2 * w], from[t][2 * w + 1], a.scale_log2, shift[t], row[t].sum);
      }
    };
    // One step: block j + 1's scores beside the probabilities of block j (scores
    // in `from`, its rows' maxima raised), then block j's product with V beside
    // the maxima of block j + 1 (into `to`). Says whether the inner loop ends: a
    // row's maximum must rise, the block needs a mask (kBreak), or there was no
    // block left (kDone, `to` not written).
    enum { kGo, kBreak, kDone };
    auto step = [&](const v16f (&from)[2], v16f (&to)[2]) __attribute__((always_inline)) -> int {
      ++j;
      if (j == j1) return kDone;
      if (!(j & 1)) enter_stage(j >> 1);
      const uint32_t at[2] = {v_at(j - 1, 0), v_at(j - 1, 1)};
      v4u vop[kAhead];
#pragma unroll
      for (int i = 0; i < kAhead; ++i) vop[i] = read_v(at, i);
      scores(j, to, [&](int i) __attribute__((always_inline)) { soften(from, i, 2 * kSteps); });
      float top[2] = {-__builtin_inff(), -__builtin_inff()};
      values(at, vop, p, [&](int i) __attribute__((always_inline)) {
#pragma unroll
        for (int u = 16 * i / (2 * kVops); u < 16 * (i + 1) / (2 * kVops); ++u)
          top[u >> 3] = fmaxf(fmaxf(top[u >> 3], to[u >> 3][2 * (u & 7)]), to[u >> 3][2 * (u & 7) + 1]);
      });
      const float m0 = max_halves(top[0]) * a.scale_log2, m1 = max_halves(top[1]) * a.scale_log2;
      const bool rise = must_raise(row[0], m0) || must_raise(row[1], m1);
      return 32 * j + 32 > clear || __builtin_amdgcn_ballot_w64(rise) != 0 ? kBreak : kGo;
    };
    enter_stage(s0);
    scores(j, s, no_slice);
    // Masks, and the rise of a row's maximum (by which what it summed so far is
    // rescaled), stay outside the inner loop: a multiply of the accumulators in
    // it makes the compiler keep a second copy of them and spill.
    for (bool more = true; more;) {
      if (32 * j + 32 > clear) mask(j, s);
      float factor[2];
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        factor[t] = raise(row[t], row_max(s[t], a.scale_log2));
        shift[t] = shift_of(row[t]);
      }
      if (__builtin_amdgcn_ballot_w64(factor[0] != 1.0f || factor[1] != 1.0f)) {
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int d = 0; d < kDims; ++d) o[t][d] *= factor[t];
      }
      for (;;) {
        int end = step(s, next);
        if (end != kGo) {
          more = end == kBreak;
          if (more) s[0] = next[0], s[1] = next[1];
          break;
        }
        end = step(next, s);
        if (end != kGo) {
          more = end == kBreak;
          if (!more) s[0] = next[0], s[1] = next[1];
          break;
        }
      }
    }
    const uint32_t at[2] = {v_at(j1 - 1, 0), v_at(j1 - 1, 1)};
    v4u vop[kAhead];
#pragma unroll
    for (int i = 0; i < kAhead; ++i) vop[i] = read_v(at, i);
    soften(s, 0, 1);
    values(at, vop, p, no_slice);
  }
  for (int stage = max(w1, s0); stage < s1; ++stage) enter_stage(stage);

  // ---- store. A lane holds dims 32 d + 8 b + 4 h + 0 .. 3 of its row; the halves
  // trade so that each stores 16 bytes.
#pragma unroll
  for (int t = 0; t < 2; ++t) {
    const float sum = sum_halves(row[t].sum);
    const bool live = 32 * t + n < wave_rows;
    const int64_t at = (q_begin + token[t]) * a.heads + head[t];
    if (a.splits > 1) {
      const int64_t part = (int64_t)split * a.q_tokens * a.heads + at;
      if (live && h == 0) a.stats[part] = split_stats(row[t].top, sum);
      if (live && sum != 0.0f) {
#pragma unroll
        for (int d = 0; d < kDims; ++d)
#pragma unroll
          for (int b = 0; b < 4; ++b)
            *reinterpret_cast<v4f*>(a.parts + part * kV + 32 * d + 8 * b + 4 * h) =
                v4f{o[t][d][4 * b], o[t][d][4 * b + 1], o[t][d][4 * b + 2], o[t][d][4 * b + 3]};
      }
      continue;
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
            w[u][e] = E::pack(o[t][d][4 * (b + u) + 2 * e] * inv, o[t][d][4 * (b + u) + 2 * e + 1] * inv);
        const auto x = __builtin_amdgcn_permlane32_swap(w[0][0], w[1][0], false, false);
        const auto y = __builtin_amdgcn_permlane32_swap(w[0][1], w[1][1], false, false);
        if (live)
          *reinterpret_cast<v4u*>(a.out + at * kV + 32 * d + 8 * (b + h)) = v4u{x[0], y[0], x[1], y[1]};
      }
  }
}

// Key splits: enough work-groups for the chip where the row tiles are few, but at
// least 256 keys to a split (a part costs 4 (d_v + 2) bytes a row, written and read).
struct PromptPlan {
  int64_t slots, splits, bytes, stats_at;
};

PromptPlan prompt_plan(int64_t q_tokens, int64_t heads, int64_t kv_heads, int64_t v_dim, int64_t sequences,
                       int64_t max_k) {
  PromptPlan p{};
  p.slots = first_slot(q_tokens, heads / kv_heads, sequences);
  const int64_t units = p.slots * kv_heads;
  const int64_t cus = device_cu_count();
  p.splits = 1;
  if (units < cus) {
    const int64_t most = (max_k + 255) / 256;
    p.splits = (2 * cus + units - 1) / units;
    if (p.splits > most) p.splits = most;
    if (p.splits > 64) p.splits = 64;
    if (p.splits < 1) p.splits = 1;
  }
  if (p.splits > 1) {
    p.stats_at = p.splits * q_tokens * heads * v_dim * 4;
    p.bytes = p.stats_at + p.splits * q_tokens * heads * 8;
  }
  return p;
}

template <typename E, int kQk, int kV>
int launch_prompt(const PromptArgs& a, hipStream_t stream) {
  hipLaunchKernelGGL((prompt_fwd<E, kQk, kV>), dim3((unsigned)((int64_t)a.slots * a.kv_heads * a.splits)), dim3(kThreads),
                     0, stream, a);
  DSA_CHECK_LAUNCH("prompt attention");
  if (a.splits > 1)
    return launch_join<E, kV>(a.parts, a.stats, a.q_tokens * a.heads, a.splits, a.cu_q, a.sequences, a.heads, a.out,
                              stream);
  return kOk;
}

template <typename E>
int launch_dims(const PromptArgs& a, int64_t qk_dim, int64_t v_dim, hipStream_t stream) {
  if (qk_dim == 192 && v_dim == 128) return launch_prompt<E, 192, 128>(a, stream);
  if (qk_dim == 128 && v_dim == 128) return launch_prompt<E, 128, 128>(a, stream);
  return launch_prompt<E, 64, 64>(a, stream);
}

}  // namespace
}  // namespace dsa

extern "C" int dsa_prompt_attention_workspace_bytes(int64_t q_tokens, int64_t heads, int64_t kv_heads, int64_t v_dim,
                                                    int64_t sequences, int64_t max_k, int64_t* bytes) {
  using namespace dsa;
  DSA_CHECK_ARG(bytes != nullptr, "null pointer");
  DSA_CHECK_ARG(q_tokens >= 0 && sequences >= 0 && max_k >= 0 && heads > 0 && kv_heads > 0 && heads % kv_heads == 0 &&
                    v_dim > 0,
                "invalid prompt attention shape");
  *bytes = prompt_plan(q_tokens, heads, kv_heads, v_dim, sequences, max_k).bytes;
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
  DSA_CHECK_ARG(heads > 0 && kv_heads > 0 && heads % kv_heads == 0 && heads <= 65536,
                "heads must be a positive multiple of kv_heads");
  DSA_CHECK_ARG(q_tokens >= 0 && k_tokens >= 0 && q_tokens < 0x7FFFFFFF && k_tokens < 0x7FFFFFFF && sequences >= 0 &&
                    sequences < 0x7FFFFFFF && max_k >= 0,
                "token and sequence counts must be in [0, 2^31)");
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
  const PromptPlan p = prompt_plan(q_tokens, heads, kv_heads, v_dim, sequences, max_k);
  DSA_CHECK_ARG(p.slots * kv_heads * p.splits < 0x7FFFFFFF, "too many row tiles");
  if (p.splits > 1)
    DSA_CHECK_ARG(workspace && reinterpret_cast<uintptr_t>(workspace) % 16 == 0 && workspace_bytes >= p.bytes,
                  "prompt attention workspace too small or misaligned");
  PromptArgs a{};
  a.q = static_cast<const uint16_t*>(q);
  a.k = static_cast<const uint16_t*>(k);
  a.v = static_cast<const uint16_t*>(v);
  a.cu_q = cu_q;
  a.cu_k = cu_k;
  a.out = static_cast<uint16_t*>(out);
  a.parts = static_cast<float*>(workspace);
  a.stats = reinterpret_cast<float2*>(static_cast<uint8_t*>(workspace) + p.stats_at);
  a.q_token = q_token_stride, a.q_head = q_head_stride;
  a.k_token = k_token_stride, a.k_head = k_head_stride;
  a.v_token = v_token_stride, a.v_head = v_head_stride;
  a.q_tokens = q_tokens, a.k_tokens = k_tokens;
  a.heads = (int32_t)heads, a.kv_heads = (int32_t)kv_heads;
  a.sequences = (int32_t)sequences, a.slots = (int32_t)p.slots, a.splits = (int32_t)p.splits;
  a.causal = causal != 0;
  a.scale_log2 = scale * kLog2E;
  return dtype == DSA_DTYPE_BF16 ? launch_dims<Bf16>(a, qk_dim, v_dim, stream)
                                 : launch_dims<F16>(a, qk_dim, v_dim, stream);
}
