// MLA attention of branches that share a long prefix, over the fp8 paged cache
// (656-byte records: 512 e4m3 latent values in 4 tiles, 4 fp32 tile scales, 64
// bf16 RoPE values; 64 tokens a page).
//
// Every query (token t of branch b, head h) attends to the whole prefix and to
// what it sees of its branch's suffix: out = sum_j p_j rec_j[:512] / sum_j p_j
// with p = exp(scale q . rec_j), in fp32 from bf16 operands (e4m3 times a power
// of two is exact in bf16; p is rounded to bf16 before the product with V).
// 2 (576 + 512) flop per (row, key).
//
// All heads read the one record of a key and the prefix is unmasked, so over the
// prefix the rows of all tokens and heads are one matrix. A work item has 128 of
// its rows, whatever branches they belong to, and a range of the keys, each record
// of which is read, converted and staged once for all 128; four waves (one per
// SIMD) take 32 rows each. With a multiple of 128 heads an item's rows are of one
// token, and its keys are the prefix and then the token's suffix; with other
// counts the suffix has items of its own, up to 128 heads of one token. Where a
// row's keys are in several items, a second launch joins their sums.
//
// A wave computes S^T = K Q^T (v_mfma_f32_32x32x16_bf16) for 32 keys and its 32
// rows, and O^T += V^T P^T with the probabilities where the scores were (the keys
// of V^T are read in the order in which a lane holds its scores). O^T takes 256 of
// a lane's 512 registers and Q^T 96 (the last 12 of its 36 operands are read from
// LDS); more rows per wave, for which an operand read would feed two products, do not
// fit. Per 32 keys a SIMD has 68 products of 32 cycles, 2.2k cycles, while the CU
// reads 320 KB of LDS and writes 37 KB, about 3.2k at 128 and 49 bytes a cycle. What
// bounds long calls is that and power: steps of 4.5k cycles ran at 2.31 GHz in 1.95 us,
// of 3.9k at 2.04 GHz in 1.92 us, and with fewer waits and scalar instructions 1.75; half
// of the LDS reads left out gave 6 %. 64 tokens of 128 heads over 65,600 keys take 940
// us, 1.24 PFLOP/s, where a library product of large matrices reaches 1.36. Short calls
// are bound by a work-group's start and end (10 us of a round) and by the parts of split
// rows (one token over 32,896 keys: 26 us and 9 for the join).
#include "attention_core.h"
#include "../../include/dsa_gfx950.h"

namespace dsa {
namespace {

constexpr int kThreads = 256;
constexpr int kQkDim = 576, kVDim = 512;
constexpr int kWaveRows = 32;
constexpr int kTileRows = 4 * kWaveRows;
constexpr int kBlockKeys = 32;
constexpr int kPageTokens = 64;
constexpr int kRecordBytes = 656;

// bf16 rows of one block in LDS: 1168 bytes = 36 dwords (mod 64) apart, so that
// 16 rows' chunks of 16 bytes, and rows r, r + 4, r + 8, r + 12 of 64 bytes, lie
// on distinct banks.
constexpr int kRowBytes = kQkDim * 2 + 16;
constexpr int kBufBytes = kBlockKeys * kRowBytes;
constexpr int kBuffers = 3;
constexpr int kSteps = kQkDim / 16, kDims = kVDim / 32;
// Q^T operands of the last kQLds steps stay in LDS, the others in registers:
// with all 36 there, O^T (256 registers of a lane) leaves too few for the rest, and
// with 28 the traded loads of Q spill some (loaded untraded they do not: long calls take
// 0.8 % less, short ones 1.4 us more).
constexpr int kQLds = 12;
constexpr int kQReg = kSteps - kQLds;
constexpr int kQBytes = kQLds * 4 * 1024;  // [wave][step][lane] 16 bytes

// A buffer's last word: 32-bit words, no swizzle.
constexpr int kRawBuffer = 0x00027000;

struct PrefixArgs {
  const uint16_t* q;
  const uint8_t* cache;
  const int32_t* prefix_table;
  const int32_t* suffix_tables;  // [branches][suffix_pages]
  const int32_t* suffix_tokens;  // [branches]
  const int32_t* cu_q;           // [branches + 1], or null: one query per branch
  uint16_t* out;
  float* parts;   // with more than one split: part_at()
  float2* stats;  // [splits][tokens * heads]
  int64_t pages, prefix;
  int32_t rows, tiles;  // tokens * heads, and their tiles
  int32_t heads, branches, suffix_pages;
  int32_t joint;  // items have the prefix and the suffix
  int32_t items, splits;                  // of the row tiles of all tokens
  int32_t suffix_splits;                  // of the suffix's own items
  float scale_log2;
};

// Key order of a score tile: row m = 16 t + 8 u + 4 h + jj holds key 16 t + 4 jj
// + 2 u + h, so that the four keys of a transposing V read are 4 rows apart.
__device__ __forceinline__ int tile_key(int m) {
  return (m & 16) + 4 * (m & 3) + 2 * ((m >> 3) & 1) + ((m >> 2) & 1);
}

template <bool kHigh>
__device__ __forceinline__ uint32_t dequant_pair(uint32_t word, float scale) {
  return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(word, scale, kHigh));
}

// Where four dims (of `dim4` fours) of a row's part begin: rows in groups of 32, a
// group's [dim4][row] as the lanes of an accumulator have them, so that a store of
// both halves is 1 KB in one piece (by rows, in pieces of 32 bytes, the stores of 128
// rows took 16k cycles).
__device__ __forceinline__ int64_t part_at(int64_t part, int64_t rows, int64_t row, int dim4) {
  const int64_t groups = (rows + 31) >> 5;
  return (((part * groups + (row >> 5)) * (kVDim / 4) + dim4) * 32 + (row & 31)) * 4;
}

__global__ __launch_bounds__(kThreads, 1) void shared_prefix_fwd(const PrefixArgs a) {
  using E = Bf16;
  __shared__ __align__(1024) uint8_t lds[kBuffers * kBufBytes + kQBytes];
  const uint32_t lds_base = (uint32_t)(uintptr_t)&lds[0];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int n = lane & 31, h = lane >> 5;
  const int all_rows = a.rows;  // (all of this in 32 bits, which hold the rows of a call)

  // ---- the item: its rows, how many keys of the prefix and of a suffix they
  // see, and its range of their blocks. Items of one range are neighbours, and
  // each XCD takes an eighth of the items in that order: they read the same
  // records from its L2.
  int row0, row_end;
  int64_t prefix = 0, suffix = 0;
  const int32_t* suffix_table = nullptr;
  int split, splits, part;
  int token = -1;  // whose suffix the item has
  if (blockIdx.x < (uint32_t)a.items) {
    const uint32_t item = (blockIdx.x & 7) * ((uint32_t)a.items >> 3) + (blockIdx.x >> 3);
    if (item >= (uint32_t)a.tiles * (uint32_t)a.splits) return;
    split = part = (int)(item / (uint32_t)a.tiles);
    splits = a.splits;
    row0 = (int)(item - (uint32_t)split * (uint32_t)a.tiles) * kTileRows;
    row_end = min(row0 + kTileRows, all_rows);
    prefix = a.prefix;
    if (a.joint) token = (int)((uint32_t)row0 / (uint32_t)a.heads);
  } else {
    const uint32_t item = blockIdx.x - (uint32_t)a.items;
    const uint32_t groups = ((uint32_t)a.heads + kTileRows - 1) / kTileRows;
    splits = a.suffix_splits;
    const uint32_t unit = item / (uint32_t)splits;
    split = (int)(item - unit * (uint32_t)splits);
    part = a.splits + split;
    token = (int)(unit / groups);
    const int head0 = (int)(unit - (uint32_t)token * groups) * kTileRows;
    row0 = token * a.heads + head0;
    row_end = token * a.heads + min(head0 + kTileRows, (int)a.heads);
  }
  // Q^T operands, in AGPRs and the last in LDS, on their way while the keys of the
  // item are looked up.
  const int wave_row = row0 + wave * kWaveRows;
  // Operands 4 g .. 4 g + 3 of half h are bytes 128 g + 64 h on of the lane's row, loaded
  // as whole 64 bytes of each of its quad's rows and traded later. (With loads of 16 bytes
  // of each of 32 rows, and divisions of 64 bits, 4.8 us went by before the first records
  // were asked for; so 2.3. One token over 32,896 keys 38.8 -> 37.4 us.)
  v4u q_ops[kQReg], q_rest[kQLds];
  static_for<4>([&](auto j) {
    const uint32_t quad_row = quad_lane<j>((uint32_t)min(wave_row + n, all_rows - 1));
    const uint16_t* src = a.q + (int64_t)quad_row * kQkDim + 32 * h + 8 * (lane & 3);
#pragma unroll
    for (int g = 0; g < kQReg / 4; ++g) q_ops[4 * g + j] = *reinterpret_cast<const v4u*>(src + 64 * g);
#pragma unroll
    for (int g = 0; g < kQLds / 4; ++g)
      q_rest[4 * g + j] = *reinterpret_cast<const v4u*>(src + 64 * (kQReg / 4 + g));
  });
  const uint32_t q_lds = lds_base + kBuffers * kBufBytes + (uint32_t)wave * (kQLds * 1024) + 16 * lane;
  __builtin_amdgcn_sched_barrier(0);

  int row_begin = row0;
  if (a.cu_q != nullptr) {
    // Rows of no branch are left alone.
    row_begin = (int)max((int64_t)row0, a.cu_q[0] * (int64_t)a.heads);
    row_end = (int)min((int64_t)row_end, a.cu_q[a.branches] * (int64_t)a.heads);
    if (row_begin >= row_end) return;
  }
  if (token >= 0) {
    int branch = token;
    int64_t left = 0;  // queries of the branch after this one
    if (a.cu_q != nullptr) {
      int lo = 0, hi = a.branches;  // the last branch that starts at or before it
      while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (a.cu_q[mid] <= token) lo = mid; else hi = mid;
      }
      branch = lo;
      left = max((int64_t)a.cu_q[lo + 1] - 1 - token, (int64_t)0);
    }
    const int64_t held = min((int64_t)a.suffix_tokens[branch], (int64_t)a.suffix_pages * kPageTokens);
    suffix = max(held - left, (int64_t)0);
    suffix_table = a.suffix_tables + (int64_t)branch * a.suffix_pages;
  }
  const int prefix_blocks = (int)((prefix + kBlockKeys - 1) / kBlockKeys);
  const int all_blocks = prefix_blocks + (int)((suffix + kBlockKeys - 1) / kBlockKeys);
  const int per_split = (all_blocks + splits - 1) / splits;
  const int b0 = split * per_split;
  const int b1 = min(b0 + per_split, all_blocks);

  const bool live = wave_row + n < row_end && wave_row + n >= row_begin;  // this lane's row, in both halves
  const int row_at = min(wave_row + n, row_end - 1);
  const bool active = __builtin_amdgcn_readfirstlane(wave_row < row_end && b1 > b0);

  // ---- staging: eight lanes a key. Lane j brings bytes 128 i + 16 j of the
  // latent (a chunk of every tile), the scales, and bytes 16 j of the RoPE part.
  const int kk = threadIdx.x >> 3, j8 = threadIdx.x & 7;
  // (Selections, not branches, in what a step needs for a block to come; blocks from b1
  // on have the last one's page, and no keys.)
  auto page_of = [&](int b) -> int {
    const int c = min(b, b1 - 1), own = c - prefix_blocks;
    return (own < 0 ? a.prefix_table : suffix_table)[(own < 0 ? c : own) >> 1];
  };
  // Valid keys of block b on `page`.
  const uint32_t pages = (uint32_t)a.pages;
  auto keys_of = [&](int b, int page) -> int {
    const int own = b - prefix_blocks;
    const int left = own < 0 ? (int)prefix - b * kBlockKeys : (int)suffix - own * kBlockKeys;
    return (b < b1) & ((uint32_t)page < pages) ? min(left, kBlockKeys) : 0;
  };
  // Its records as a buffer that ends with them: what lies behind reads as zeros, so
  // that what a masked key's p = 0 multiplies is finite.
  auto records_of = [&](int b, int page, int keys) {
    const int half = (b < prefix_blocks ? b : b - prefix_blocks) & 1;
    const int64_t row = (int64_t)(keys > 0 ? page : 0) * kPageTokens + half * kBlockKeys;
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(a.cache + row * kRecordBytes), 0,
                                             keys * kRecordBytes, kRawBuffer);
  };
  typedef v4u Staged[6];
  const int fetch_lane = kk * kRecordBytes + 16 * j8, scale_lane = kk * kRecordBytes + kVDim;
  // Vector i of the staged ones: chunks 0 .. 3, the scales, the RoPE part.
  auto fetch = [&](Staged& st, auto records, int i) __attribute__((always_inline)) {
    st[i] = __builtin_bit_cast(v4u, __builtin_amdgcn_raw_buffer_load_b128(
        records, i == 4 ? scale_lane : fetch_lane + (i == 5 ? kVDim + 16 : 128 * i), 0, 0));
  };
  // Part u of the landed record: half u & 1 of chunk u / 2 as bf16 (word by word, of
  // which `words` of one call are converted), from u = 8 on the RoPE part.
  v4u converted;
  auto unpack = [&](const Staged& st, uint32_t to, int u, int from, int words) __attribute__((always_inline)) {
    if (u == 8) {
      lds_store<v4u>(to + 2 * kVDim - 16 * j8, st[5]);
      return;
    }
    const float scale = __builtin_bit_cast(v4f, st[4])[u >> 1];
#pragma unroll
    for (int w = from; w < from + words; ++w) {
      const uint32_t codes = st[u >> 1][2 * (u & 1) + w];
      converted[2 * w] = dequant_pair<false>(codes, scale);
      converted[2 * w + 1] = dequant_pair<true>(codes, scale);
    }
    if (from + words == 2) lds_store<v4u>(to + 256 * (u >> 1) + 16 * (u & 1), converted);
  };
  const uint32_t store_lane = (uint32_t)kk * kRowBytes + 32 * j8;
  // Buffers go round: the one after `at` (an address within it).
  auto after = [&](uint32_t at) -> uint32_t {
    return at + kBufBytes >= lds_base + kBuffers * kBufBytes ? at + kBufBytes - kBuffers * kBufBytes : at + kBufBytes;
  };

  v16f o[kDims];
  RowState row{-__builtin_inff(), 0.0f};

  // LDS lane addresses. K: key tile_key(n), dims 64 (ks / 4) + 32 h + 8 (ks % 4). V: lane 4 jj + qq
  // of 16-lane group g reads key 16 t + 4 jj + 2 u + h, dims 32 d + 16 (g & 1) + 4 qq.
  const uint32_t k_lane = (uint32_t)tile_key(n) * kRowBytes + 64 * h;
  const uint32_t v_lane = (uint32_t)(4 * ((lane & 15) >> 2) + h) * kRowBytes + 32 * ((lane >> 4) & 1) + 8 * (lane & 3);
  constexpr int kAhead = 3, kVops = 2 * kDims;

  auto read_v = [&](uint32_t at, int i) __attribute__((always_inline)) -> v4u {
    const int t = i & 1, d = i >> 1;
    const v2u lo = lds_column(at + (16 * t) * kRowBytes + 64 * d);
    const v2u hi = lds_column(at + (16 * t + 2) * kRowBytes + 64 * d);
    return v4u{lo.x, lo.y, hi.x, hi.y};
  };
  constexpr auto k_step = [](int ks) { return 128 * (ks >> 2) + 16 * (ks & 3); };
  static_assert(kQReg % 4 == 0 && kQLds % 4 == 0, "operands in fours");
  v4u kop[kAhead];
  auto read_first_k = [&](uint32_t buffer) __attribute__((always_inline)) -> uint32_t {
    const uint32_t at = opaque(buffer + k_lane);
#pragma unroll
    for (int ks = 0; ks < kAhead; ++ks) kop[ks] = lds_load<v4u>(at + k_step(ks));
    return at;
  };
  // S of a block at `at`, whose first kAhead operands are in kop.
  auto scores = [&](uint32_t at, v16f& s, auto slice) __attribute__((always_inline)) {
    v4u qop[2];
    s = v16f{};
#pragma unroll
    for (int ks = 0; ks < kSteps; ++ks) {
      s = E::mfma(kop[ks % kAhead], ks < kQReg ? q_ops[ks < kQReg ? ks : 0] : qop[ks & 1], s);
      if (ks + kAhead < kSteps) kop[ks % kAhead] = lds_load<v4u>(at + k_step(ks + kAhead));
      if (ks + 2 >= kQReg && ks + 2 < kSteps) qop[ks & 1] = lds_load<v4u>(q_lds + 1024 * (ks + 2 - kQReg));
      slice(ks);
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  // Products from .. to - 1 of the block at `at` with V.
  auto values = [&](uint32_t at, v4u (&vop)[kAhead], const v4u (&p)[2], int from, int to, auto slice)
                    __attribute__((always_inline)) {
#pragma unroll
    for (int i = from; i < to; ++i) {
      o[i >> 1] = E::mfma(vop[i % kAhead], p[i & 1], o[i >> 1]);
      if (i + kAhead < kVops) vop[i % kAhead] = read_v(at, i + kAhead);
      slice(i);
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  auto mask = [&](int seen, v16f& s) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < 16; ++i) s[i] = tile_key(8 * (i >> 2) + 4 * h + (i & 3)) < seen ? s[i] : -__builtin_inff();
  };

  // ---- pipeline. Step b: scores of block b + 1 beside the probabilities of
  // block b, then block b's product with V beside the conversion of block b + 2
  // into LDS; block b + 3's records are on their way. One barrier per step; three
  // buffers.
  // Valid keys of blocks b, b + 1 and b + 2; the page of block b + 3.
  int keys, keys1, keys2, page3 = -1;
  Staged st;
  {
    // The first two blocks on their way together.
    int page = -1, page1 = -1, page2 = -1;
    if (b1 > b0) page = page_of(b0), page1 = page_of(b0 + 1), page2 = page_of(b0 + 2), page3 = page_of(b0 + 3);
    keys = keys_of(b0, page), keys1 = keys_of(b0 + 1, page1), keys2 = keys_of(b0 + 2, page2);
    Staged first;
    const auto from = records_of(b0, page, keys), from1 = records_of(b0 + 1, page1, keys1),
               from2 = records_of(b0 + 2, page2, keys2);
#pragma unroll
    for (int i = 0; i < 6; ++i) fetch(first, from, i);
#pragma unroll
    for (int i = 0; i < 6; ++i) fetch(st, from1, i);
#pragma unroll
    for (int g = 0; g < kQLds / 4; ++g) transpose_quad(&q_rest[4 * g]);
#pragma unroll
    for (int ks = 0; ks < kQLds; ++ks) lds_store<v4u>(q_lds + 1024 * ks, q_rest[ks]);
#pragma unroll
    for (int g = 0; g < kQReg / 4; ++g) transpose_quad(&q_ops[4 * g]);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int u = 0; u < 9; ++u) unpack(first, lds_base + store_lane, u, 0, 2);
#pragma unroll
    for (int u = 0; u < 9; ++u) unpack(st, lds_base + kBufBytes + store_lane, u, 0, 2);
#pragma unroll
    for (int i = 0; i < 6; ++i) fetch(st, from2, i);
  }
  // On to the next block: block b + 3's records, whose page is asked for a step ahead.
  auto advance = [&](int b) {
    const int page = __builtin_amdgcn_readfirstlane(page3);
    const int keys3 = keys_of(b + 3, page);
    const auto from = records_of(b + 3, page, keys3);
    page3 = page_of(b + 4);
    keys = keys1, keys1 = keys2, keys2 = keys3;
    return from;
  };
#pragma unroll
  for (int ks = 0; ks < kQReg; ++ks) asm volatile("" : "+a"(q_ops[ks]));
  lds_barrier();
#pragma unroll
  for (int d = 0; d < kDims; ++d) o[d] = v16f{};
  if (active) {
    int b = b0;
    v16f s, next;
    v4u p[2];
    float shift = 0.0f;
    auto no_slice = [](int) {};
    Softener<E> softener;
    constexpr int kPairs = 8, kTicks = kPairs + 2;
    auto soften = [&](const v16f& from, int i, int of) __attribute__((always_inline)) {
#pragma unroll
      for (int u = kTicks * i / of; u < kTicks * (i + 1) / of; ++u)
        softener.tick(u, kPairs, a.scale_log2, [&](int e) { return from[e]; }, &shift, [&](int w, uint32_t pair) {
          p[w >> 2][w & 3] = pair;
          row.sum = E::add_pair(pair, row.sum);
        });
    };
    enum { kGo, kBreak, kDone };
    uint32_t now = lds_base;  // block b's buffer
    uint32_t k_now = read_first_k(now);
    auto step = [&](const v16f& from, v16f& to) __attribute__((always_inline)) -> int {
      if (b + 1 == b1) return kDone;
      const auto from3 = advance(b);
      ++b;
      const uint32_t at = opaque(now + v_lane);
      now = after(now);
      v4u vop[kAhead];
      scores(k_now, to, [&](int i) __attribute__((always_inline)) {
        soften(from, i, kSteps);
        if (i >= kSteps - kAhead) vop[i - (kSteps - kAhead)] = read_v(at, i - (kSteps - kAhead));
      });
      // Computed by here, beside the products, not where they are used.
      asm volatile("" : "+v"(p[0]), "+v"(p[1]), "+v"(row.sum));
      const uint32_t ahead = after(now);
      const uint32_t store = opaque(ahead + store_lane);
      float top = -__builtin_inff();
      // Two words of a record converted at a time, and its place taken by the next.
      values(at, vop, p, 0, kVops - kAhead, [&](int i) __attribute__((always_inline)) {
        if (i < 16) unpack(st, store, i >> 1, i & 1, 1);
        if (i == 16) unpack(st, store, 8, 0, 2);
        if (i % 4 == 0 && i > 0 && i <= 16) fetch(st, from3, i / 4 - 1);
        if (i == 18) fetch(st, from3, 5);
        if (i == 20) fetch(st, from3, 4);
        if (i >= 8 && i < 16) top = fmaxf(fmaxf(top, to[2 * (i - 8)]), to[2 * (i - 8) + 1]);
      });
      // The last products' operands are in registers: the next block's first are read
      // beside them.
      lds_barrier();
      k_now = read_first_k(ahead);
      const float mx = max_halves(top) * a.scale_log2;
      const uint64_t rise = __builtin_amdgcn_ballot_w64(must_raise<E>(row, mx));
      values(at, vop, p, kVops - kAhead, kVops, no_slice);
      return keys < kBlockKeys || rise != 0 ? kBreak : kGo;
    };
    scores(k_now, s, no_slice);
    k_now = read_first_k(after(now));
    for (bool more = true; more;) {
      if (keys < kBlockKeys) mask(keys, s);
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
    const uint32_t at = opaque(now + v_lane);
    v4u vop[kAhead];
#pragma unroll
    for (int i = 0; i < kAhead; ++i) vop[i] = read_v(at, i);
    soften(s, 0, 1);
    values(at, vop, p, 0, kVops, no_slice);
  } else {
    // A wave without rows stages its keys all the same.
    uint32_t to = lds_base + 2 * kBufBytes;
    for (int b = b0; b + 1 < b1; ++b, to = after(to)) {
      const auto from3 = advance(b);
#pragma unroll
      for (int u = 0; u < 9; ++u) unpack(st, to + store_lane, u, 0, 2);
#pragma unroll
      for (int i = 0; i < 6; ++i) fetch(st, from3, i);
      lds_barrier();
    }
  }

  // ---- store (as in prompt attention: the halves trade to store 16 bytes).
  const float sum = sum_halves(row.sum);
  if (a.splits + a.suffix_splits > 1) {
    if (live && h == 0) a.stats[(int64_t)part * all_rows + row_at] = split_stats(row.top, sum);
    if (live && sum != 0.0f) {
      float* to = a.parts + part_at(part, all_rows, row_at, h);
#pragma unroll
      for (int d = 0; d < kDims; ++d)
#pragma unroll
        for (int c = 0; c < 4; ++c)
          *reinterpret_cast<v4f*>(to + (8 * d + 2 * c) * 128) =
              v4f{o[d][4 * c], o[d][4 * c + 1], o[d][4 * c + 2], o[d][4 * c + 3]};
    }
    return;
  }
  const float inv = sum > 0.0f ? 1.0f / sum : (sum == 0.0f ? 0.0f : sum);
#pragma unroll
  for (int d = 0; d < kDims; ++d)
#pragma unroll
    for (int c = 0; c < 4; c += 2) {
      uint32_t w[2][2];
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int e = 0; e < 2; ++e)
          w[u][e] = E::pack(o[d][4 * (c + u) + 2 * e] * inv, o[d][4 * (c + u) + 2 * e + 1] * inv);
      const auto x = __builtin_amdgcn_permlane32_swap(w[0][0], w[1][0], false, false);
      const auto y = __builtin_amdgcn_permlane32_swap(w[0][1], w[1][1], false, false);
      if (live) *reinterpret_cast<v4u*>(a.out + (int64_t)row_at * kVDim + 32 * d + 8 * (c + h)) = v4u{x[0], y[0], x[1], y[1]};
    }
}

// Joins the parts of the rows: a wave has four dims (a lane's 16 bytes) of 32 rows in
// each half, kChunks waves neighbouring ones, and kWays of them every kWays-th part
// each, four in flight at a time, against a running maximum of their own. What bounds
// it is reading the parts (171 of 128 rows, 45 MB: 9.9 us).
template <int kWays, int kChunks>
__global__ __launch_bounds__(64 * kWays * kChunks) void join_parts(
    const float* __restrict__ parts, const float2* __restrict__ stats, int64_t rows, int splits,
    const int32_t* __restrict__ cu, int32_t branches, int64_t heads, uint16_t* __restrict__ out) {
  __shared__ v4f shared[kWays][kChunks][64];
  __shared__ float2 of_way[kWays][32];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int way = wave % kWays, chunk = wave / kWays;
  constexpr int kPerGroup = kVDim / 8 / kChunks;  // work-groups of 32 rows
  const int64_t row = (int64_t)(blockIdx.x / kPerGroup) * 32 + (lane & 31);
  const int dim4 = 2 * ((int)(blockIdx.x % kPerGroup) * kChunks + chunk) + (lane >> 5);
  const float none = -__builtin_inff();
  // Rows outside the branches have no parts, and stay as they are.
  const bool live = row < rows && (cu == nullptr || (row >= cu[0] * heads && row < cu[branches] * heads));
  v4f acc = {};
  float top = none, sum = 0.0f;
  if (live) {
    constexpr int kAtOnce = 4;
    for (int s0 = way; s0 < splits; s0 += kWays * kAtOnce) {
      float2 st[kAtOnce];
      v4f o[kAtOnce];
#pragma unroll
      for (int i = 0; i < kAtOnce; ++i) {
        const int s = s0 + i * kWays;
        st[i] = s < splits ? stats[s * rows + row] : make_float2(none, 0.0f);
        o[i] = s < splits ? *reinterpret_cast<const v4f*>(parts + part_at(s, rows, row, dim4)) : v4f{};
      }
      float up = top;
#pragma unroll
      for (int i = 0; i < kAtOnce; ++i) up = fmaxf(up, st[i].x);
      const float keep = top == none ? 0.0f : __builtin_amdgcn_exp2f(top - up);
      sum *= keep;
      acc *= keep;
#pragma unroll
      for (int i = 0; i < kAtOnce; ++i) {
        // (A part without a visible key has no values in memory. A NaN maximum, of
        // one with a NaN score, spreads.)
        if (st[i].y == 0.0f) continue;
        const float w = __builtin_amdgcn_exp2f(st[i].x - up);
        sum += w * st[i].y;
        acc += w * o[i];
      }
      top = up;
    }
  }
  if constexpr (kWays > 1) {
    shared[way][chunk][lane] = acc;
    if (chunk == 0 && lane < 32) of_way[way][lane] = make_float2(top, sum);
    __syncthreads();
    if (way != 0) return;
#pragma unroll
    for (int w = 1; w < kWays; ++w) top = fmaxf(top, of_way[w][lane & 31].x);
    sum = 0.0f;
    acc = v4f{};
#pragma unroll
    for (int w = 0; w < kWays; ++w) {
      const float2 st = of_way[w][lane & 31];
      if (st.y == 0.0f) continue;
      const float factor = st.x == none ? st.y : __builtin_amdgcn_exp2f(st.x - top);
      sum += factor * st.y;
      acc += factor * shared[w][chunk][lane];
    }
  }
  if (!live) return;
  const float inv = sum > 0.0f ? 1.0f / sum : (sum == 0.0f ? 0.0f : sum);
  *reinterpret_cast<v2u*>(out + row * kVDim + 4 * dim4) =
      v2u{Bf16::pack(acc.x * inv, acc.y * inv), Bf16::pack(acc.z * inv, acc.w * inv)};
}

// Ways for the parts there are (14 parts of 2,048 rows: 11.0 us with 2, 13.6 with 4; 91
// of 256: 10.9 and 9.0); 16 where the rows alone do not fill the chip (171 of 128: 9.9 us,
// with 4 12.3).
int join_ways(int64_t rows, int64_t splits) { return splits <= 4 ? 1 : splits <= 32 ? 2 : rows >= 256 ? 4 : 16; }

int launch_join_parts(const PrefixArgs& a, int64_t rows, int splits, hipStream_t stream) {
  const auto go = [&](auto kernel, int ways, int chunks) {
    hipLaunchKernelGGL(kernel, dim3((unsigned)((rows + 31) / 32 * (kVDim / 8 / chunks))), dim3(64 * ways * chunks), 0,
                       stream, a.parts, a.stats, rows, splits, a.cu_q, a.branches, (int64_t)a.heads, a.out);
  };
  const int ways = join_ways(rows, splits);
  if (ways == 1) go(join_parts<1, 4>, 1, 4);
  else if (ways == 2) go(join_parts<2, 4>, 2, 4);
  else if (ways == 4) go(join_parts<4, 2>, 4, 2);
  else go(join_parts<16, 1>, 16, 1);
  DSA_CHECK_LAUNCH("join of the shared prefix's parts");
  return kOk;
}

// Key splits: the count of least time, by the rounds of work-groups (one per CU),
// their fixed part, the steps of the longest, and what writing a row's parts and
// reading them again costs. Fitted to one token of 128 heads over 32,896 keys (103,
// 147, 206 splits: 38.0, 36.6, 36.0 us), 18 over 10,330 (11, 14: 78, 75), 30 over 572 (1,
// 2, 4, 6: 41, 34, 30, 34), 114 over 528 (1, 2, 3: 42, 51, 70) and 8 over 70,000 (16, 32,
// 64: 294, 164, 231).
constexpr double kFixedUs = 10.0, kStepUs = 1.75, kJoinUs = 3.0, kPartUsPerRow = 0.0007;

struct PrefixPlan {
  bool joint;
  int64_t splits, suffix_splits, stats_at, bytes;
};

PrefixPlan prefix_plan(int64_t tokens, int64_t heads, int64_t prefix, int64_t suffix_pages) {
  PrefixPlan p{};
  const int64_t cus = device_cu_count();
  const int64_t rows = tokens * heads;
  if (rows == 0) return p;
  const int64_t prefix_blocks = (prefix + kBlockKeys - 1) / kBlockKeys;
  const int64_t suffix_blocks = suffix_pages * (kPageTokens / kBlockKeys);
  p.joint = heads % kTileRows == 0;
  // Work-groups and blocks of a split of the first kind of items, and of the
  // suffix's own.
  const int64_t tiles = (rows + kTileRows - 1) / kTileRows;
  const int64_t blocks = p.joint ? prefix_blocks + suffix_blocks : prefix_blocks;
  const int64_t own_tiles = tokens * ((heads + kTileRows - 1) / kTileRows);
  const bool first = p.joint || prefix > 0, own = !p.joint && (suffix_pages > 0 || prefix == 0);
  double least = 1e30;
  for (int64_t ss = own ? 1 : 0; ss <= (own ? 64 : 0) && (ss <= 1 || ss <= suffix_blocks); ss *= 2) {
    static constexpr int kSteps1[] = {1, 2, 3, 4, 5, 6, 8, 10, 12, 16};
    for (int64_t r = 0; r <= 12 + 10; ++r) {
      // One; or as many as some rounds hold, with or without the suffix's own items;
      // or splits of a few blocks: at most one per block, and no more than give the
      // same longest split.
      int64_t s = first ? 1 : 0;
      if (first && r > 0) {
        s = r > 12 ? (blocks + kSteps1[r - 13] - 1) / kSteps1[r - 13]
                   : r % 2 ? (r + 1) / 2 * cus / tiles : (r / 2 * cus - own_tiles * ss) / tiles;
        if (s > 256) s = 256;
        if (s > blocks) s = blocks;
        if (s < 1) continue;
        s = (blocks + (blocks + s - 1) / s - 1) / ((blocks + s - 1) / s);
      }
      // Rounds of the first kind, and of the suffix's own items, which come last, as
      // far as the CUs that the last of those rounds leaves free do not take them.
      const int64_t full = (tiles * s + cus - 1) / cus, room = full * cus - tiles * s;
      const double step = s > 0 ? kFixedUs + kStepUs * (double)((blocks + s - 1) / s) : 0.0;
      const double own_step = ss > 0 ? kFixedUs + kStepUs * (double)((suffix_blocks + ss - 1) / ss) : 0.0;
      const int64_t rest = ss > 0 ? own_tiles * ss - room * (int64_t)(step / own_step + 0.5) : 0;
      double us = (double)full * step + (rest > 0 ? (double)((rest + cus - 1) / cus) * own_step : 0.0);
      if (us < own_step) us = own_step;
      if (s + ss > 1) us += kJoinUs + kPartUsPerRow * (double)(rows * (s + ss));
      if (us < least) {
        least = us;
        p.splits = s;
        p.suffix_splits = ss;
      }
    }
    if (ss == 0) break;
  }
  const int64_t parts = p.splits + p.suffix_splits;
  if (parts > 1) {
    p.stats_at = parts * ((rows + 31) / 32 * 32) * kVDim * 4;
    p.bytes = p.stats_at + parts * rows * 8;
  }
  return p;
}

// What the plan's and the kernel's arithmetic is made for.
int check_sizes(int64_t tokens, int64_t heads, int64_t prefix_tokens, int64_t suffix_pages) {
  DSA_CHECK_ARG(tokens >= 0 && heads > 0 && heads <= 65536, "invalid shared prefix MLA shape");
  DSA_CHECK_ARG(prefix_tokens >= 0 && prefix_tokens < 0x7FFFFFFF && suffix_pages >= 0 &&
                    suffix_pages < 0x7FFFFFFF / kPageTokens,
                "prefix and suffix lengths must fit int32");
  DSA_CHECK_ARG(tokens < (0x7FFFFF00 + heads - 1) / heads, "too many query rows");
  return kOk;
}

}  // namespace
}  // namespace dsa

extern "C" int dsa_shared_prefix_mla_workspace_bytes(int64_t tokens, int64_t heads, int64_t prefix_tokens,
                                                     int64_t suffix_pages, int64_t* bytes) {
  using namespace dsa;
  DSA_CHECK_ARG(bytes != nullptr, "null pointer");
  if (const int status = check_sizes(tokens, heads, prefix_tokens, suffix_pages); status != kOk) return status;
  *bytes = prefix_plan(tokens, heads, prefix_tokens, suffix_pages).bytes;
  return kOk;
}

extern "C" int dsa_shared_prefix_mla_fp8(const void* q, int64_t tokens, int64_t heads, const void* cache,
                                         int64_t pages, const int32_t* prefix_table, int64_t prefix_tokens,
                                         const int32_t* suffix_tables, int64_t suffix_pages,
                                         const int32_t* suffix_tokens, const int32_t* cu_q, int64_t branches,
                                         float scale, void* out, void* workspace, int64_t workspace_bytes,
                                         hipStream_t stream) {
  using namespace dsa;
  DSA_CHECK_ARG(branches >= 0 && branches < 0x7FFFFFFF, "invalid shared prefix MLA shape");
  if (const int status = check_sizes(tokens, heads, prefix_tokens, suffix_pages); status != kOk) return status;
  DSA_CHECK_ARG(scale > 0.0f && __builtin_isfinite(scale), "scale must be positive and finite");
  if (tokens == 0) return kOk;
  DSA_CHECK_ARG(branches > 0 && (cu_q != nullptr || branches == tokens),
                "without cu_q every branch has one query");
  DSA_CHECK_ARG(pages >= 1 && pages < 0x7FFFFFFF / kPageTokens, "cache rows must fit int32");
  DSA_CHECK_ARG(q && cache && out && suffix_tokens && (prefix_tokens == 0 || prefix_table) &&
                    (suffix_pages == 0 || suffix_tables),
                "null pointer");
  DSA_CHECK_ARG((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(cache) | reinterpret_cast<uintptr_t>(out)) %
                        16 == 0,
                "q, cache and out must be 16-byte aligned");
  const PrefixPlan p = prefix_plan(tokens, heads, prefix_tokens, suffix_pages);
  const int64_t tiles = (tokens * heads + kTileRows - 1) / kTileRows;
  const int64_t items = p.splits > 0 ? (tiles * p.splits + 7) / 8 * 8 : 0;
  const int64_t own = tokens * ((heads + kTileRows - 1) / kTileRows) * p.suffix_splits;
  // (The join has a wave for each way and eight dims of 32 rows.)
  const int64_t rows = tokens * heads, joined = p.bytes > 0 ? join_ways(rows, p.splits + p.suffix_splits) : 0;
  DSA_CHECK_ARG(grid_fits(items + own, kThreads) && grid_fits((rows + 31) / 32 * (kVDim / 8) * joined, 64),
                "too many query rows");
  if (p.bytes > 0)
    DSA_CHECK_ARG(workspace && reinterpret_cast<uintptr_t>(workspace) % 16 == 0 && workspace_bytes >= p.bytes,
                  "shared prefix MLA workspace too small or misaligned");
  PrefixArgs a{};
  a.q = static_cast<const uint16_t*>(q);
  a.cache = static_cast<const uint8_t*>(cache);
  a.prefix_table = prefix_table;
  a.suffix_tables = suffix_tables;
  a.suffix_tokens = suffix_tokens;
  a.cu_q = cu_q;
  a.out = static_cast<uint16_t*>(out);
  a.parts = static_cast<float*>(workspace);
  a.stats = reinterpret_cast<float2*>(static_cast<uint8_t*>(workspace) + p.stats_at);
  a.rows = (int32_t)(tokens * heads), a.tiles = (int32_t)tiles;
  a.pages = pages, a.prefix = prefix_tokens;
  a.heads = (int32_t)heads, a.branches = (int32_t)branches, a.suffix_pages = (int32_t)suffix_pages;
  a.joint = p.joint, a.items = (int32_t)items, a.splits = (int32_t)p.splits;
  a.suffix_splits = (int32_t)p.suffix_splits;
  a.scale_log2 = scale * kLog2E;
  hipLaunchKernelGGL(shared_prefix_fwd, dim3((unsigned)(items + own)), dim3(kThreads), 0, stream, a);
  DSA_CHECK_LAUNCH("shared prefix MLA");
  if (p.bytes > 0) return launch_join_parts(a, rows, (int)(p.splits + p.suffix_splits), stream);
  return kOk;
}
