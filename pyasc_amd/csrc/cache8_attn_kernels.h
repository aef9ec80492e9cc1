// Attention over a cache held in 8 bits: the device code of asc_quantized_cache_attention.
//
// The queries that share a key / value head are its rows: row r is query r % n of the head's query head r / n.
// With codes c and a scale per block, k_j = ks_j ck_j and v_j = vs_j cv_j, so
//   s_j = (q . ck_j) (sm_scale ks_j),   o = sum_j (p_j vs_j) cv_j / sum_j p_j,   p_j = exp(s_j - m):
// the codes go to the matrix units as they are, in fp16, which holds all of them exactly, K's scales go into the
// scores' factor and V's into the probabilities.  A tile has 64 keys, of 16 of which each group lies in one
// block and one page, so a lane has four factors per tile.  P^T's values are e_j = 2^-M p_j vs_j, with a reference point M of
// their own that follows the row's largest s_j + log2 vs_j as m follows its largest s_j: V scales may lie as far apart as fp32
// holds, and keys that a row does not attend, or with next to no probability, have no say in it.  exp2 takes log2 vs_j with the
// scores' shift, and a group's sum of e_j times 2^(M - m) / vs_j is its part of the denominator.  A row's scale that lies 2^-60
// and more below its 2^(M - m) counts as that: blocks of zeros, with scales of 2^-126, have their share of the denominator.
// Queries of bf16 are brought to fp16's range by a power of two of their row: exact down to 2^-31 of its largest element, and to
// 2^-39 of that below.
//
// The e_j are rounded to fp16 for the product with the values, as matrix operands have to be (2^-11 of each, and below 2^-22 of a
// row's largest 2^-33 of that): errors of up to 0.0002 of the results' norm, beside 0.0017 of a bf16 result's own rounding.
// Beside 0.0002 of an fp16 result's they count where a few keys outweigh the rest (0.0003 in all, one row over 500 keys): the
// kernel for few rows, whose matrix units wait for the cache, multiplies what the rounding leaves as a second term (0.0002; 8
// sequences of up to 32768 keys take 74.6 us for 72.3).
#pragma once

#include "cache8.h"
#include "flash_attn_kernels.h"
#include "kv_attn_kernels.h"

namespace asc {
namespace c8 {

using fa::BKV;
using fa::F16;
using fa::f32x16;
using fa::lds_addr;
using fa::other_half;
using kv::f32x4;

constexpr int kGroup = 16, kGroups = BKV / kGroup;

struct AttnArgs {
  Cache c;
  const uint16_t* q;
  uint16_t* o;
  float* lse;  // [batch, q_heads, n] or null
  int64_t q_batch, q_head, q_seq, o_batch, o_head, o_seq;  // elements
  float* part_o;   // [unit][rows][D], unnormalised, in units of 2^M
  float* part_ml;  // [unit][rows][4]: m, sum of the probabilities in units of 2^m, M
  int32_t batch, group, rows, row_blocks, splits, join_groups, causal;
  int32_t lanes, per_lane;  // of the order of the row blocks
  uint32_t units;  // batch * splits * kv_heads
  Divisor by_n, by_heads, by_splits, by_slots, by_lanes;
  // sm_scale log2(e) as a mantissa, which goes into K's scales, and a power of two, which goes with the queries': neither product
  // leaves fp32 where the scores do not.
  float scale_mantissa;
  int32_t scale_power;

  // Tiles of a split of `total` tiles: the last splits may have none.
  __device__ __forceinline__ int per(int total) const { return static_cast<int>(by_splits.divide(total + splits - 1)); }
};

// Four codes of a word as two packed pairs of fp16.
template <class Q>
__device__ __forceinline__ u32x2 codes_to_f16(uint32_t w) {
  typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
  if constexpr (__is_same(Q, Int8)) {
    // 1024 + (c + 128) has c + 128 as its lowest bits
    w ^= 0x80808080u;
    const f16x2 lift = {static_cast<_Float16>(1152.0f), static_cast<_Float16>(1152.0f)};
    const f16x2 lo = __builtin_bit_cast(f16x2, __builtin_amdgcn_perm(0x64646464u, w, 0x04010400u)) - lift;
    const f16x2 hi = __builtin_bit_cast(f16x2, __builtin_amdgcn_perm(0x64646464u, w, 0x04030402u)) - lift;
    return u32x2{__builtin_bit_cast(uint32_t, lo), __builtin_bit_cast(uint32_t, hi)};
  } else {
    const auto lo = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, false);
    const auto hi = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, true);
    return u32x2{__builtin_bit_cast(uint32_t, lo), __builtin_bit_cast(uint32_t, hi)};
  }
}
template <class Q>
__device__ __forceinline__ u32x4 operand_of(uint32_t lo, uint32_t hi) {
  const u32x2 a = codes_to_f16<Q>(lo), b = codes_to_f16<Q>(hi);
  return u32x4{a[0], a[1], b[0], b[1]};
}

// One workgroup's share, as kv::Share.  Causal: the row blocks with most keys first, which are the last ones of each of the
// group's heads (`lanes` runs of per_lane blocks).
__device__ __forceinline__ kv::Share share_of(const AttnArgs& p) {
  const uint32_t slot = blockIdx.x >> 3;
  const uint32_t per = p.by_slots.divide(slot), place = slot - per * p.by_slots.d;
  const uint32_t back = p.by_lanes.divide(place), run = place - back * p.lanes;
  kv::Share s;
  s.unit = per * 8 + (blockIdx.x & 7);
  s.row0 = static_cast<int>(run + 1) * p.per_lane - 1 - static_cast<int>(back);
  s.live = s.unit < p.units && s.row0 < p.row_blocks;
  const uint32_t range = p.by_heads.divide(s.unit);
  s.head = static_cast<int>(s.unit - range * p.c.kv_heads);
  s.b = static_cast<int>(p.by_splits.divide(range));
  s.split = static_cast<int>(range - static_cast<uint32_t>(s.b) * p.splits);
  return s;
}

// What a sequence has: its keys, and its queries among n.
struct Sequence {
  int len, news, first;  // query i attends the first min(first + i, len) keys
  bool bad;
  __device__ __forceinline__ Sequence(const AttnArgs& p, int b) {
    bad = false;
    len = kv::clamped(p.c.lengths[b], p.c.capacity, bad);
    news = kv::clamped(p.c.news ? p.c.news[b] : p.c.n, p.c.n, bad);
    first = p.causal ? len - news + 1 : len;
  }
  __device__ __forceinline__ int limit(int query) const { return min(max(first + query, 0), len); }
};
// Queries of sequence b that are written (more than n: all of them, as NaN).
__device__ __forceinline__ int written_of(const AttnArgs& p, int b) { return p.c.news ? p.c.news[b] : p.c.n; }

// The most keys that a row of row0 .. row0 + rows - 1 attends.
__device__ __forceinline__ int limit_of_rows(const AttnArgs& p, const Sequence& s, int row0, int rows) {
  const int last = min(row0 + rows, p.rows) - 1;
  const int g = p.by_n.divide(row0);
  const int query = static_cast<int>(p.by_n.divide(last)) == g ? last - g * p.c.n : p.c.n - 1;
  const int q = min(query, s.news - 1);
  return q < 0 ? 0 : s.limit(q);
}

// The fewest keys that a row of row0 .. row0 + rows - 1 with a query attends.
__device__ __forceinline__ int least_of_rows(const AttnArgs& p, const Sequence& s, int row0, int rows) {
  const int last = min(row0 + rows, p.rows) - 1;
  const int g = p.by_n.divide(row0), query = row0 - g * p.c.n;
  // the first row's, where they are of one head; else a head's first query is among them
  if (static_cast<int>(p.by_n.divide(last)) == g) return query < s.news ? s.limit(query) : s.len;
  return s.news > 0 ? s.limit(0) : s.len;
}

// Output row `row` of the share, false where nothing is written.
__device__ __forceinline__ bool out_row(const AttnArgs& p, const kv::Share& s, int row, int written, int64_t& o_at,
                                        int64_t& lse_at) {
  if (row >= p.rows) return false;
  const int g = p.by_n.divide(row), query = row - g * p.c.n;
  if (query >= written) return false;
  const int64_t head = s.head * p.group + g;
  o_at = s.b * p.o_batch + head * p.o_head + query * p.o_seq;
  lse_at = (static_cast<int64_t>(s.b) * p.c.kv_heads * p.group + head) * p.c.n + query;
  return true;
}

// This lane's row: its elements, and its query (-1: none).  kPairs: lane half h holds columns 32 t + 16 h + 0..15 in
// operands 2 t and 2 t + 1 (as K's codes are read), else 16 k + 8 h + 0..7 in operand k.
template <int D, bool kPairs>
__device__ __forceinline__ int load_query(const AttnArgs& p, const kv::Share& s, int row, int h, u32x4 (&q)[D / 16]) {
  const int r = min(row, p.rows - 1), g = p.by_n.divide(r), query = r - g * p.c.n;
  const uint16_t* at = p.q + s.b * p.q_batch + static_cast<int64_t>(s.head * p.group + g) * p.q_head + query * p.q_seq;
#pragma unroll
  for (int k = 0; k < D / 16; ++k) {
    const int column = kPairs ? (k >> 1) * 32 + h * 16 + (k & 1) * 8 : k * 16 + h * 8;
    q[k] = *reinterpret_cast<const u32x4*>(at + column);
  }
  return row < p.rows ? query : -1;
}
// The keys that it attends (a row without a query restricts nothing), its elements in fp16 and its scores' power of two.
template <int D, class E>
__device__ __forceinline__ void take_query(const AttnArgs& p, const Sequence& seq, int query, u32x4 (&q)[D / 16], int& limit,
                                           int& power) {
  const bool any = query >= 0 && query < seq.news;
  limit = any ? seq.limit(query) : seq.len;
  power = p.scale_power;
#pragma unroll
  for (int k = 0; k < D / 16; ++k) q[k] = any ? q[k] : u32x4{0, 0, 0, 0};
  if constexpr (__is_same(E, fa::Bf16)) {
    uint32_t most = 0;
#pragma unroll
    for (int k = 0; k < D / 16; ++k)
#pragma unroll
      for (int w = 0; w < 4; ++w) most = max(most, max(q[k][w] & 0x7fffu, q[k][w] >> 16 & 0x7fffu));
    most = max(most, __float_as_uint(other_half(__uint_as_float(most))));
    // the largest lands in [2^14, 2^15)
    const uint32_t exponent = max(most >> 7, 14u);
    const int up = exponent == 255 ? 0 : 141 - static_cast<int>(exponent);
    const float scale = __uint_as_float(static_cast<uint32_t>(127 + up) << 23);
    power -= up;
#pragma unroll
    for (int k = 0; k < D / 16; ++k)
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        q[k][w] = F16::pack(__uint_as_float(q[k][w] << 16) * scale, __uint_as_float(q[k][w] & 0xffff0000u) * scale);
      }
  }
}

// What a wave knows of its tiles' groups: sixteen of its tiles at a time, whose 64 groups its lanes work out together, lane 4 t + g
// group g of tile first + t * step.  The next sixteen's entries of the table and scales are asked for on the way
// (kEntries, kScales), as their use waits for all loads before it.
constexpr int kBatch = 64 / kGroups, kEntries = 4, kScales = 8;

struct Groups {
  uint32_t k0, v0, ks0, vs0;  // the sequence's head
  const int32_t* table;       // null: one piece
  int len, b, lane, step;
  int first;                  // of the current tiles
  bool poison;                // a page or a length outside the cache: the rows' results are NaN
  uint32_t k, v;              // places of the groups' first rows, units of 16 bytes
  float ks, vs;               // scales (K's times scale_mantissa), 0 behind the last key
  uint32_t next_id, next_k, next_v;
  float next_ks, next_vs;

  __device__ __forceinline__ void init(const AttnArgs& p, const kv::Share& s, int lane_, int step_) {
    k0 = s.head * p.c.ks.head;
    v0 = s.head * p.c.vs.head;
    ks0 = s.head * p.c.kss.head;
    vs0 = s.head * p.c.vss.head;
    table = p.c.table ? p.c.table + s.b * p.c.table_stride : nullptr;
    b = s.b;
    lane = lane_;
    step = step_;
  }
  __device__ __forceinline__ int key_of(int from) const {
    return (from + (lane / kGroups) * step) * BKV + (lane % kGroups) * kGroup;
  }
  // The entries of the table for the tiles from `from` on; a length that is not known yet is taken for the capacity.
  __device__ __forceinline__ uint32_t entries(const AttnArgs& p, int from, int end) const {
    const int key = key_of(from);
    return table && key < end ? static_cast<uint32_t>(table[p.c.page.divide(key)]) : 0;
  }
  // Groups behind the last key are read as their tile's first, and those of tiles behind it not at all.
  __device__ __forceinline__ void places(const AttnArgs& p, int from, uint32_t id, uint32_t& at_k, uint32_t& at_v, float& s_k,
                                         float& s_v) {
    const int key = key_of(from);
    const bool there = key < len;
    const uint32_t row = key - p.c.page.divide(key) * p.c.page.d;
    if (!table) id = b;
    const bool bad = there && id >= p.c.pages;
    poison = poison || __builtin_amdgcn_ballot_w64(bad) != 0;
    if (bad) id = 0;
    s_k = s_v = 0.f;
    at_k = at_v = 0;
    if (there) {
      const uint32_t block = p.c.block.divide(row);
      at_k = k0 + id * p.c.ks.page + row * p.c.ks.row;
      at_v = v0 + id * p.c.vs.page + row * p.c.vs.row;
      s_k = p.c.k_scale[ks0 + id * p.c.kss.page + block * p.c.kss.row] * p.scale_mantissa;
      s_v = p.c.v_scale[vs0 + id * p.c.vss.page + block * p.c.vss.row];
    }
    // lane 0 of each four: its tile's first
    const uint32_t tile_k = __builtin_amdgcn_mov_dpp(static_cast<int>(at_k), 0x00, 0xF, 0xF, true);
    const uint32_t tile_v = __builtin_amdgcn_mov_dpp(static_cast<int>(at_v), 0x00, 0xF, 0xF, true);
    at_k = there ? at_k : tile_k;
    at_v = there ? at_v : tile_v;
  }
  __device__ __forceinline__ void start(const AttnArgs& p, int from, uint32_t id) {
    first = from;
    places(p, from, id, k, v, ks, vs);
  }
  // Before tile number t of the current ones (end: keys of the tiles that are worked on).
  __device__ __forceinline__ void ask(const AttnArgs& p, int t, int end) {
    const int from = first + kBatch * step;
    if (t == kEntries && from * BKV < end) next_id = entries(p, from, len);
    if (t == kScales && from * BKV < end) places(p, from, next_id, next_k, next_v, next_ks, next_vs);
  }
  // To the next tiles, where number n is the first of them.
  __device__ __forceinline__ void advance(int& n) {
    const bool on = n == kBatch;
    first += on ? kBatch * step : 0;
    k = on ? next_k : k;
    v = on ? next_v : v;
    ks = on ? next_ks : ks;
    vs = on ? next_vs : vs;
    n = on ? 0 : n;
  }
  // Place of group g of tile number t, of these tiles or the next.
  template <bool kIsV>
  __device__ __forceinline__ uint32_t place(int t, int g) const {
    const uint32_t now = __builtin_amdgcn_readlane(kIsV ? v : k, (t * kGroups + g) & 63);
    const uint32_t next = __builtin_amdgcn_readlane(kIsV ? next_v : next_k, (t * kGroups + g) & 63);
    return t < kBatch ? now : next;
  }
};

constexpr float kLeast = 60.0f;  // a row's 2^(M - m) over the least V scale that counts, log2

// The online softmax of a wave: lane (row, half h of the keys); register r of score block kb is key 32 kb + 8 (r / 4) +
// 4 h + r % 4, of group 2 kb + r / 8.
template <int D>
struct Softmax {
  static constexpr int kDBlocks = D / 32;
  f32x16 acc[kDBlocks];  // in units of 2^M
  float m, M;            // reference points (log2): of the scores, and of the scores plus log2 of the V scale
  float l;               // this lane half's sum of the probabilities in units of 2^m
  int power;             // of the raw scores, beside K's scales
  int limit;             // keys of the row
  float log_scale;       // of this lane's group: log2 of the V scale
  float a[kGroups];      // of the tile's groups: the factors of their scores,
  float log_v[kGroups];  // and log2 of the V scale

  __device__ __forceinline__ void init() {
#pragma unroll
    for (int i = 0; i < kDBlocks; ++i) acc[i] = f32x16{};
    m = M = -INFINITY;
    l = 0.f;
  }
  // The V scales of the current tiles, one per lane.  What is not positive counts as 2^-160, whose values round to zero.
  __device__ __forceinline__ void take_scales(float vs) {
    const bool small = vs < 0x1p-100f;  // the logarithm takes no subnormal numbers
    log_scale = fmaxf(__builtin_amdgcn_logf(small ? vs * 0x1p64f : vs) - (small ? 64.0f : 0.0f), -160.0f);
  }
  // Those of tile number t, and its K scales.
  __device__ __forceinline__ void set_tile(float ks, int t) {
    const auto lane = [&](float v, int g) {
      return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), t * kGroups + g));
    };
#pragma unroll
    for (int g = 0; g < kGroups; ++g) {
      // not zero, which times the -inf of a hidden key would be NaN
      a[g] = fmaxf(ldexpf(lane(ks, g), power), 0x1p-126f);
      log_v[g] = lane(log_scale, g);
    }
  }
  __device__ __forceinline__ void hide(f32x16 (&s)[2], int j, int h) const {
#pragma unroll
    for (int kb = 0; kb < 2; ++kb)
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        if (j * BKV + kb * 32 + (r >> 2) * 8 + h * 4 + (r & 3) >= limit) s[kb][r] = -INFINITY;
      }
  }
  // The largest score of half kb of a tile, or of all of it, and the largest with its V scale, less fp16's lift.
  struct Tops {
    float m, M;
  };
  __device__ __forceinline__ Tops half_tops(const f32x16& s, int kb) const {
    float low = -INFINITY, high = -INFINITY;
#pragma unroll
    for (int r = 0; r < 8; ++r) {
      low = fmaxf(low, s[r]);
      high = fmaxf(high, s[8 + r]);
    }
    low *= a[kb * 2];
    high *= a[kb * 2 + 1];
    const float top = fmaxf(low, high), with_v = fmaxf(low + log_v[kb * 2], high + log_v[kb * 2 + 1]);
    return {fmaxf(top, other_half(top)) - F16::kLift, fmaxf(with_v, other_half(with_v)) - F16::kLift};
  }
  __device__ __forceinline__ Tops tile_tops(const f32x16 (&s)[2]) const {
    const Tops x = half_tops(s[0], 0), y = half_tops(s[1], 1);
    return {fmaxf(x.m, y.m), fmaxf(x.M, y.M)};
  }
  // Of a row's first tile.
  __device__ __forceinline__ void start(const Tops& top) {
    m = top.m;
    M = top.M;
  }
  __device__ __forceinline__ void raise(const Tops& top) {
    const bool up = top.m > m, up_v = top.M > M;
    l *= up ? __builtin_amdgcn_exp2f(m - top.m) : 1.0f;
    const float alpha = up_v ? __builtin_amdgcn_exp2f(M - top.M) : 1.0f;
    if (up) m = top.m;
    if (up_v) M = top.M;
#pragma unroll
    for (int i = 0; i < kDBlocks; ++i) acc[i] *= alpha;
  }
  // What the probabilities are taken against: the reference points, and the least log2 of a V scale that counts.
  struct Reference {
    float m, M, least;
  };
  __device__ __forceinline__ Reference reference() const {
    return m == -INFINITY ? Reference{0.f, 0.f, -kLeast} : Reference{m, M, M - m - kLeast};
  }
  // The scores' shift of group g, and the factor from e_j to p_j.
  __device__ __forceinline__ float shift_of(const Reference& r, int g) const { return fmaxf(log_v[g], r.least) - r.M; }
  __device__ __forceinline__ float undo_of(const Reference& r, int g) const { return __builtin_amdgcn_exp2f(-r.m - shift_of(r, g)); }
  // Sums of a lane over a half, or a whole tile: of the probabilities, and of P^T's values.
  struct Sums {
    float p, e;
  };
  // Values 2 w and 2 w + 1 of group u of half kb, and their sum.
  __device__ __forceinline__ void pair(const f32x16& s, int kb, int u, int w, const Reference& ref, u32x4 (&pb)[2], float& sum) const {
    const int g = kb * 2 + u;
    const float e0 = __builtin_amdgcn_exp2f(fmaf(s[8 * u + 2 * w], a[g], shift_of(ref, g)));
    const float e1 = __builtin_amdgcn_exp2f(fmaf(s[8 * u + 2 * w + 1], a[g], shift_of(ref, g)));
    sum += e0;
    sum += e1;
    pb[u][w] = F16::pack(e0, e1);
  }
  __device__ __forceinline__ void add_group(Sums& sums, const Reference& ref, int g, float sum) const {
    sums.p = fmaf(sum, undo_of(ref, g), sums.p);
    sums.e += sum;
  }
  // P^T operands of half kb.
  __device__ __forceinline__ Sums probs(const f32x16& s, int kb, u32x4 (&pb)[2]) const {
    const Reference ref = reference();
    Sums sums{0.f, 0.f};
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      float sum = 0.f;
#pragma unroll
      for (int w = 0; w < 4; ++w) pair(s, kb, u, w, ref, pb, sum);
      add_group(sums, ref, kb * 2 + u, sum);
    }
    return sums;
  }
  // The values may not overflow fp16; and where the probabilities grow as far, what counts as the least scale would.
  __device__ __forceinline__ bool out_of_range(const Sums& sums) const {
    return __builtin_amdgcn_ballot_w64(fmaxf(sums.p, sums.e) > F16::kTileSumLimit || m == -INFINITY) != 0;
  }
  __device__ __forceinline__ void guard(const f32x16& s, int kb, u32x4 (&pb)[2], Sums sums) {
    if (out_of_range(sums)) {
      raise(half_tops(s, kb));
      sums = probs(s, kb, pb);
    }
    l += sums.p;
  }
  // kRest: and what their rounding leaves, rounded.
  template <bool kRest>
  __device__ __forceinline__ Sums both_probs(const f32x16 (&s)[2], u32x4 (&pb)[2][2], u32x4 (&rest)[2][2]) const {
    if constexpr (!kRest) {
      const Sums x = probs(s[0], 0, pb[0]), y = probs(s[1], 1, pb[1]);
      return {x.p + y.p, x.e + y.e};
    }
    const Reference ref = reference();
    Sums sums{0.f, 0.f};
#pragma unroll
    for (int g = 0; g < kGroups; ++g) {
      float sum = 0.f;
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        const int r = 8 * (g & 1) + 2 * w;
        const float e0 = __builtin_amdgcn_exp2f(fmaf(s[g >> 1][r], a[g], shift_of(ref, g)));
        const float e1 = __builtin_amdgcn_exp2f(fmaf(s[g >> 1][r + 1], a[g], shift_of(ref, g)));
        sum += e0;
        sum += e1;
        const uint32_t x = F16::pack(e0, e1);
        const fa::f16x2 rounded = __builtin_bit_cast(fa::f16x2, x);
        pb[g >> 1][g & 1][w] = x;
        rest[g >> 1][g & 1][w] = F16::pack(e0 - static_cast<float>(rounded[0]), e1 - static_cast<float>(rounded[1]));
      }
      add_group(sums, ref, g, sum);
    }
    return sums;
  }
  template <bool kRest>
  __device__ __forceinline__ void tile_probs(const f32x16 (&s)[2], u32x4 (&pb)[2][2], u32x4 (&rest)[2][2]) {
    Sums sums = both_probs<kRest>(s, pb, rest);
    if (out_of_range(sums)) {
      raise(tile_tops(s));
      sums = both_probs<kRest>(s, pb, rest);
    }
    l += sums.p;
  }
  // A NaN among the values of keys that only some rows attend is taken as zero in the products, whose 0 times NaN
  // would reach all rows (without_nan).  Where that was met, the rows that attend it get it back: tile j, from memory.
  __device__ __forceinline__ void add_nan(const AttnArgs& p, const kv::Share& s, int j, int h) {
    for (int i = 0; i < BKV; ++i) {
      const int key = j * BKV + i;
      uint32_t page, row;
      if (__builtin_amdgcn_ballot_w64(key < limit) == 0) return;
      if (!place(p.c, s.b, key, page, row)) continue;  // NaN already
      const uint8_t* v = p.c.v + row_at(p.c.vs, page, s.head, row) + h * 4;
#pragma unroll
      for (int db = 0; db < kDBlocks; ++db)
#pragma unroll
        for (int rq = 0; rq < 4; ++rq) {
          const uint32_t w = *reinterpret_cast<const uint32_t*>(v + db * 32 + rq * 8);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            if (key < limit && (w >> (8 * e) & 0x7fu) == 0x7fu) acc[db][rq * 4 + e] = __builtin_nanf("");
          }
        }
    }
  }
};

// A word of e4m3 codes with zeros in place of NaN, noted in `found`.
__device__ __forceinline__ uint32_t without_nan(uint32_t w, uint32_t& found) {
  const uint32_t nan = ((w & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u;
  found |= nan;
  return w & ~((nan >> 7) * 0xffu);
}

// ------------------------------------------------------------------------------------ few rows
//
// Bound by the cache's bytes: 64 sequences of 1024 to 4096 keys (8 heads of 128 columns, int8) are 335 MB in 66 us, 5.1 TB/s with the
// start and the last sequences' end, 6.0 between (a plain copy: 6.1); one token of each costs nothing beside them.  A wave
// works on tiles of its own, without barriers, with the next tile's K and V on their way to LDS in the meantime.

template <int D>
struct Narrow {
  static constexpr int kWaves = 4, kWgPerCu = D == 128 ? 2 : 3;
  static constexpr int kRows = 32;
  static constexpr int kTile = BKV * D;           // bytes
  static constexpr int kLoads = kTile / 1024;     // of a wave
  static constexpr int kRowsPerLoad = 1024 / D;
};

// One wave's tiles: codes in LDS as they are, in 16-byte chunks whose place in a row is flipped by the row so that 16
// rows' reads of a chunk (K) and a transposing read's eight rows (V) lie in different banks.
template <int D, class Q>
struct NarrowTiles {
  using N = Narrow<D>;
  static constexpr int kChunks = D / 16;
  uint8_t* k;
  uint8_t* v;
  int lane, col, h;
  uint32_t kaddr, vaddr;
  uint32_t koff[2], voff[2];

  static __device__ __forceinline__ int kflip(int row) { return D == 128 ? (row >> 1) & 7 : (row >> 2) & 3; }
  static __device__ __forceinline__ int vflip(int row) {
    return D == 128 ? ((row >> 1) & 1) * 2 + ((row >> 3) & 1) * 4 : ((row >> 3) & 1) * 2;
  }
  __device__ __forceinline__ void init(const AttnArgs& p) {
    kaddr = lds_addr(k) + col * D + ((h ^ kflip(col)) << 4);
    // lane 2 i + half of a group of 16 reads half a chunk of row i; lane i receives column i of eight rows
    const int i = (lane & 15) >> 1, row = h * 4 + (i & 3) + (i >> 2) * 8;
    vaddr = lds_addr(v) + row * D + ((((lane >> 4) & 1) ^ vflip(row)) << 4) + (lane & 1) * 8;
#pragma unroll
    for (int odd = 0; odd < 2; ++odd) {
      const int in_group = (D == 128 ? odd * 8 : 0) + lane / kChunks, pos = lane % kChunks;
      koff[odd] = in_group * p.c.ks.row * 16 + ((pos ^ kflip(in_group)) << 4);
      voff[odd] = in_group * p.c.vs.row * 16 + ((pos ^ vflip(in_group)) << 4);
    }
  }
  // Tile number t of the current ones or the next.
  template <bool kIsV>
  __device__ __forceinline__ void load(const AttnArgs& p, const Groups& groups, int t) const {
    const uint64_t base = reinterpret_cast<uint64_t>(kIsV ? p.c.v : p.c.k);
    uint8_t* dst = kIsV ? v : k;
#pragma unroll
    for (int i = 0; i < N::kLoads; ++i) {
      const uint32_t place = groups.template place<kIsV>(t, D == 128 ? i >> 1 : i);
      const uint8_t* src = reinterpret_cast<const uint8_t*>(base + static_cast<uint64_t>(place) * 16);
      const uint32_t off = kIsV ? voff[i & 1] : koff[i & 1];
      __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)(src + off),
                                       (__attribute__((address_space(3))) void*)(dst + i * 1024), 16, 0, 0);
    }
  }
  // Raw scores of the tile.
  __device__ __forceinline__ void scores(const u32x4 (&q)[D / 16], f32x16 (&s)[2]) const {
    constexpr int kPairs = D / 32, kReads = 2 * kPairs, kWin = 4;
    u32x4 x[kReads];
#pragma unroll
    for (int r = 0; r < kWin && r < kReads; ++r) x[r] = fa::lds_read_b128(kaddr ^ ((r % kPairs) << 5), r / kPairs * 32 * D);
    s[0] = f32x16{};
    s[1] = f32x16{};
#pragma unroll
    for (int r = 0; r < kReads; ++r) {
      fa::lds_wait(x[r], r + kWin <= kReads ? kWin - 1 : kReads - 1 - r);
      const u32x4 lo = operand_of<Q>(x[r][0], x[r][1]), hi = operand_of<Q>(x[r][2], x[r][3]);
      if (r + kWin < kReads) {
        x[r + kWin] = fa::lds_read_b128(kaddr ^ (((r + kWin) % kPairs) << 5), (r + kWin) / kPairs * 32 * D);
      }
      f32x16& t = s[r / kPairs];
      t = F16::mfma(lo, q[r % kPairs * 2], t);
      t = F16::mfma(hi, q[r % kPairs * 2 + 1], t);
    }
  }
  static __device__ __forceinline__ u32x2 read_tr(uint32_t addr, int off) {
    u32x2 r;
    asm volatile("ds_read_b64_tr_b8 %0, %1 offset:%2" : "=v"(r) : "v"(addr), "i"(off));
    return r;
  }
  static __device__ __forceinline__ void wait(u32x2& r, int n) { asm volatile("s_waitcnt lgkmcnt(%1)" : "+v"(r) : "i"(n)); }
  // Operand r: block r / 4 of the columns, keys 16 (r % 4) .. + 15.
  template <bool kMasked, bool kRest>
  __device__ __forceinline__ void pv(Softmax<D>& st, const u32x4 (&pb)[2][2], const u32x4 (&rest)[2][2], uint32_t& found) const {
    constexpr int kOps = 4 * (D / 32), kWin = 8;
    u32x2 x[kOps];
#pragma unroll
    for (int r = 0; r < kWin; ++r) x[r] = read_tr(vaddr ^ ((r >> 2) << 5), (r & 3) * 16 * D);
#pragma unroll
    for (int r = 0; r < kOps; ++r) {
      wait(x[r], r + kWin <= kOps ? kWin - 1 : kOps - 1 - r);
      if constexpr (kMasked) x[r] = u32x2{without_nan(x[r][0], found), without_nan(x[r][1], found)};
      const u32x4 a = operand_of<Q>(x[r][0], x[r][1]);
      if (r + kWin < kOps) x[r + kWin] = read_tr(vaddr ^ (((r + kWin) >> 2) << 5), (r & 3) * 16 * D);
      st.acc[r >> 2] = F16::mfma(a, pb[(r & 3) >> 1][r & 1], st.acc[r >> 2]);
      if constexpr (kRest) st.acc[r >> 2] = F16::mfma(a, rest[(r & 3) >> 1][r & 1], st.acc[r >> 2]);
    }
  }
};

// What brings sums of values in units of 2^M over one of probabilities in units of 2^m to a result: a factor, and a power of two
// behind it, as their product may lie outside fp32.
struct Result {
  float factor;
  int power;
  __device__ __forceinline__ Result(float m, float M, float l) {
    const float apart = m == -INFINITY ? 0.f : fminf(fmaxf(M - m, -400.0f), 400.0f), whole = floorf(apart);
    factor = kv::inverse_sum(l) * __builtin_amdgcn_exp2f(apart - whole);
    power = static_cast<int>(whole);
  }
  __device__ __forceinline__ float of(float x) const { return ldexpf(x * factor, power); }
};

// Waves' parts in LDS, or a row's splits, joined and written: eight values of row `row`, relative to their largest
// reference points m and M.
template <class E>
__device__ __forceinline__ void write_row(const AttnArgs& p, const kv::Share& s, int row, int ch, float (&o)[8], float m, float M,
                                          float l, int written) {
  int64_t o_at, lse_at;
  if (!out_row(p, s, row, written, o_at, lse_at)) return;
  const Result result(m, M, l);
#pragma unroll
  for (int e = 0; e < 8; ++e) o[e] = result.of(o[e]);
  *reinterpret_cast<u32x4*>(p.o + o_at + ch * 8) = kv::pack8<E>(o, 1.0f);
  if (p.lse != nullptr && ch == 0) p.lse[lse_at] = kv::lse_of(m, l);
}

// Up to 32 rows; the workgroup's four waves take every fourth tile each.
template <int D, class E, class Q>
__device__ __forceinline__ void narrow_body(const AttnArgs& p) {
  using N = Narrow<D>;
  constexpr int kWaves = N::kWaves, L = N::kLoads, kRow = D * 4;
  constexpr bool kHasNan = __is_same(Q, E4m3);
  constexpr bool kRest = __is_same(E, F16);
  static_assert(N::kRows * kRow <= 2 * BKV * D, "a wave's part reuses its tiles");
  __shared__ __attribute__((aligned(256))) uint8_t lds[kWaves * 2 * N::kTile];
  __shared__ float stats[3][kWaves][N::kRows];

  kv::Share s = share_of(p);
  if (!s.live) return;
  s.row0 *= N::kRows;
  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  NarrowTiles<D, Q> t;
  t.lane = tid & 63;
  t.col = t.lane & 31;
  t.h = t.lane >> 5;
  t.k = lds + wave * 2 * N::kTile;
  t.v = t.k + N::kTile;
  t.init(p);
  // what does not wait for the sequence's length is asked for with it
  Groups groups;
  groups.init(p, s, t.lane, kWaves);
  u32x4 q[D / 16];
  const int query = load_query<D, true>(p, s, s.row0 + t.col, t.h, q);
  uint32_t id = 0;
  if (p.splits == 1) id = groups.entries(p, wave, p.c.capacity);
  const Sequence seq(p, s.b);
  groups.len = seq.len;
  groups.poison = seq.bad;
  Softmax<D> st;
  st.init();

  const int total = (limit_of_rows(p, seq, s.row0, N::kRows) + BKV - 1) / BKV;
  const int per = p.per(total);
  const int begin = min(total, s.split * per), end = min(total, begin + per);
  int j = begin + wave;
  if (j < end) {
    if (p.splits > 1) id = groups.entries(p, j, groups.len);
    groups.start(p, j, id);
    t.template load<false>(p, groups, 0);
    t.template load<true>(p, groups, 0);
  }
  take_query<D, E>(p, seq, query, q, st.limit, st.power);
  int least = st.limit;  // keys that all rows attend
#pragma unroll
  for (int d = 1; d < 32; d *= 2) least = min(least, __shfl_xor(least, d, 64));
  least = __builtin_amdgcn_readfirstlane(least);
  uint32_t found = 0;
  for (int n = 0; j < end; j += kWaves, ++n) {  // tile number n of the current ones
    const bool next = j + kWaves < end;
    if (n == 0 || n == kBatch) {
      groups.advance(n);
      st.take_scales(groups.vs);
    }
    // all but V_j have landed
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"(L) : "memory");
    f32x16 sc[2];
    t.scores(q, sc);
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    if (next) t.template load<false>(p, groups, n + 1);
    st.set_tile(groups.ks, n);
    const bool masked = (j + 1) * BKV > least;
    if (masked) st.hide(sc, j, t.h);
    if (j == begin + wave) st.start(st.tile_tops(sc));  // nothing to rescale yet
    u32x4 pb[2][2], rest[2][2];
    st.template tile_probs<kRest>(sc, pb, rest);
    if (next) {
      asm volatile("s_waitcnt vmcnt(%0)" ::"n"(L) : "memory");  // all but the next tile's K
    } else {
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    }
    if (kHasNan && masked) {
      t.template pv<true, kRest>(st, pb, rest, found);
    } else {
      t.template pv<false, kRest>(st, pb, rest, found);
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    groups.ask(p, n, end * BKV);
    if (next) t.template load<true>(p, groups, n + 1);
  }
  if (kHasNan && __builtin_amdgcn_ballot_w64(found != 0) != 0) {
    for (int i = begin + wave; i < end; i += kWaves) {
      if ((i + 1) * BKV > least) st.add_nan(p, s, i, t.h);
    }
  }

  // the waves' parts, relative to their own reference points, through LDS
  const auto part_off = [](int row, int c) { return row * kRow + ((c ^ (row & 15)) << 4); };
  {
    float l = st.l + other_half(st.l);
    if (groups.poison) l = __builtin_nanf("");
    if (t.h == 0) {
      stats[0][wave][t.col] = st.m;
      stats[1][wave][t.col] = l;
      stats[2][wave][t.col] = st.M;
    }
#pragma unroll
    for (int db = 0; db < D / 32; ++db)
#pragma unroll
      for (int rq = 0; rq < 4; ++rq) {
        const f32x16& a = st.acc[db];
        *reinterpret_cast<f32x4*>(t.k + part_off(t.col, db * 8 + rq * 2 + t.h)) =
            f32x4{a[rq * 4], a[rq * 4 + 1], a[rq * 4 + 2], a[rq * 4 + 3]};
      }
  }
  __syncthreads();
  const int written = written_of(p, s.b);
#pragma unroll
  for (int i = 0; i < N::kRows * (D / 8) / (kWaves * 64); ++i) {
    const int cc = tid + kWaves * 64 * i;
    const int row = cc / (D / 8), ch = cc % (D / 8);
    if (s.row0 + row >= p.rows) continue;
    float m = stats[0][0][row], M = stats[2][0][row];
#pragma unroll
    for (int w = 1; w < kWaves; ++w) {
      m = fmaxf(m, stats[0][w][row]);
      M = fmaxf(M, stats[2][w][row]);
    }
    float f[kWaves], l_run = 0.f;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      const float mw = stats[0][w][row], Mw = stats[2][w][row];
      l_run += (mw == m ? 1.0f : __builtin_amdgcn_exp2f(mw - m)) * stats[1][w][row];
      f[w] = Mw == M ? 1.0f : __builtin_amdgcn_exp2f(Mw - M);
    }
    float o[8] = {};
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      const uint8_t* part = lds + w * 2 * N::kTile;
      const f32x4 lo = *reinterpret_cast<const f32x4*>(part + part_off(row, 2 * ch));
      const f32x4 hi = *reinterpret_cast<const f32x4*>(part + part_off(row, 2 * ch + 1));
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        o[e] = fmaf(f[w], lo[e], o[e]);
        o[4 + e] = fmaf(f[w], hi[e], o[4 + e]);
      }
    }
    if (p.splits > 1) {
      const int64_t place = static_cast<int64_t>(s.unit) * p.rows + s.row0 + row;
      if (ch == 0) *reinterpret_cast<f32x4*>(p.part_ml + place * 4) = f32x4{m, l_run, M, 0.f};
      *reinterpret_cast<f32x4*>(p.part_o + place * D + ch * 8) = f32x4{o[0], o[1], o[2], o[3]};
      *reinterpret_cast<f32x4*>(p.part_o + place * D + ch * 8 + 4) = f32x4{o[4], o[5], o[6], o[7]};
      continue;
    }
    write_row<E>(p, s, s.row0 + row, ch, o, m, M, l_run, written);
  }
}

// ------------------------------------------------------------------------------------ many rows
//
// Bound by what the waves issue: 2 sequences of 8192 keys and 2048 new rows (32 query heads on 8, 128 columns: 481 GF) in
// 465 to 475 us, 1.02 PF (a large product of matrices: 1.21), with the matrix units busy for 46% of the time, the VALU for 54%
// (a quarter of it exp2) and LDS for 29%: matrix and vector instructions follow one another, at 1.8 to 2.0 GHz.  With 64 columns
// a tile has the same exponentials for half of the products: 324 us, matrix units 31%, VALU 67%.  V scales in units of one value
// for all rows took 457 to 466 and 312 us, and lost the values of rows whose scales lie 2^-22 and more below it.
// Half a tile's probabilities are computed between the products of the halves around it (620 us without that), and what a
// tile's groups need is worked out for sixteen tiles at a time.

template <int D>
struct Wide {
  static constexpr int kWaves = D == 128 ? 8 : 4, kWgPerCu = D == 128 ? 1 : 2;
  static constexpr int kRows = 32 * kWaves;
  static constexpr int kTile = BKV * D * 2;  // bytes, in fp16
};

// Each wave loads the codes of 1024 / D rows of a tile, a piece of 16 per lane, and writes them as fp16 to LDS, where
// all waves read them.
template <int D, class E, class Q>
struct WideState : fa::FaState<D, Wide<D>::kWaves, 1, F16, true> {
  using Base = fa::FaState<D, Wide<D>::kWaves, 1, F16, true>;
  static constexpr int T = Wide<D>::kTile;
  Softmax<D> st;
  Groups groups;
  uint32_t koff, voff;        // of this lane's piece in its group of rows
  uint32_t kdst, vdst;        // of its first chunk of fp16 in a tile; the second's differs by one bit
  int group;                  // of this wave's rows
  uint32_t found;             // NaN among the values that this lane has loaded, of tiles that not all rows attend

  // Where a chunk of eight values lies in a tile: a row's second half (D 64: every other row) has neighbours swapped, since eight
  // lanes write every other chunk of 256 bytes at a time, 128 bytes of banks.
  static __device__ __forceinline__ uint32_t swapped(int row, int chunk) {
    return static_cast<uint32_t>(D == 128 ? chunk >> 3 & 1 : row & 1) << 4;
  }
  static __device__ __forceinline__ uint32_t k_place(int row, int chunk) { return fa::k_off<D>(row, chunk) ^ swapped(row, chunk); }
  static __device__ __forceinline__ uint32_t v_place(int row, int col) { return fa::v_off<D>(row, col) ^ swapped(row, col >> 3); }
  __device__ __forceinline__ void init_tiles(const AttnArgs& p) {
    constexpr int kPieces = D / 16;
    const int lane = this->lane, row = this->wave * (64 / kPieces) + lane / kPieces, piece = lane % kPieces;
    group = row / kGroup;
    koff = (row % kGroup) * p.c.ks.row * 16 + piece * 16;
    voff = (row % kGroup) * p.c.vs.row * 16 + piece * 16;
    kdst = k_place(row, piece * 2);
    vdst = v_place(row, piece * 16);
    group = __builtin_amdgcn_readfirstlane(group);
    this->kaddr[0] = k_place(this->col, this->h);
    const int g_lane = lane & 15;
    this->vaddr[0] = v_place(this->h * 4 + (g_lane >> 2), ((lane >> 4) & 1) * 16 + (g_lane & 3) * 4);
  }
  __device__ __forceinline__ u32x4 load(const uint8_t* codes, uint32_t place, uint32_t off) const {
    return *reinterpret_cast<const u32x4*>(codes + static_cast<uint64_t>(place) * 16 + off);
  }
  template <bool kClean>
  __device__ __forceinline__ void store(uint8_t* tile, uint32_t dst, u32x4 x) {
    if constexpr (kClean) {
#pragma unroll
      for (int i = 0; i < 4; ++i) x[i] = without_nan(x[i], found);
    }
    *reinterpret_cast<u32x4*>(tile + dst) = operand_of<Q>(x[0], x[1]);
    *reinterpret_cast<u32x4*>(tile + (dst ^ 16)) = operand_of<Q>(x[2], x[3]);
  }
  // V^T operand r of half kb of a tile in stage kStage: block r / 2 of the columns, its keys 16 (r % 2) .. + 15.
  template <int kStage>
  __device__ __forceinline__ u32x4 v_operand(uint32_t at, int kb, int r) const {
    const int off = kStage * T + (kb * 32 + (r & 1) * 16) * (D * 2);
    const auto lo = fa::lds_read_tr16_b64(at, off), hi = fa::lds_read_tr16_b64(at, off + 8 * (D * 2));
    return u32x4{lo[0], lo[1], hi[0], hi[1]};
  }
  // Where it lies in a tile at `base`; that of K operand r, chunks 2 r and 2 r + 1 of its rows.
  __device__ __forceinline__ uint32_t v_at(uint32_t base, int r) const {
    return (base + this->vaddr[0]) ^ (r >> 1 << 6) ^ swapped(0, (r >> 1) * 4);
  }
  __device__ __forceinline__ uint32_t k_at(uint32_t base, int r) const {
    return (base + this->kaddr[0]) ^ (r << 5) ^ swapped(0, r * 2);
  }
  template <int kStage>
  __device__ __forceinline__ u32x4 k_operand(uint32_t at, int kb, int r) const {
    return fa::lds_read_b128(at, kStage * T + kb * 32 * (D * 2));
  }
  uint32_t kat[Base::kKSteps], vat[Base::kDBlocks];  // of the operands in stage 0
  __device__ __forceinline__ void init_places(uint8_t* ring) {
#pragma unroll
    for (int r = 0; r < Base::kKSteps; ++r) kat[r] = k_at(lds_addr(ring), r);
#pragma unroll
    for (int i = 0; i < Base::kDBlocks; ++i) vat[i] = v_at(lds_addr(ring + 3 * T), 2 * i);
  }
  static constexpr int kOps = Base::kKSteps;  // of K, and as many of V, for a half of a tile
  static_assert(kOps == 2 * Base::kDBlocks, "operands of a half");

  // The probabilities of half kb (s[kb], into pb_out) between the products that wait for nothing of it: the raw scores of
  // the half behind it (into s[1 - kb], of K's stage kK) and, kPv, the values times the probabilities of the half before it
  // (pb_in, of V's stage kV).  Returns the sums of the probabilities and of their values.
  template <int kb, bool kPv, int kK, int kV>
  __device__ __forceinline__ typename Softmax<D>::Sums half(f32x16 (&s)[2], const u32x4 (&pb_in)[2], u32x4 (&pb_out)[2]) {
    constexpr int kWin = 3, kPer = 8 / kOps, kEach = kPv ? 3 : 1;  // LDS reads in a round
    const auto ref = st.reference();
    typename Softmax<D>::Sums sums{0.f, 0.f};
    float sum = 0.f;
    u32x4 x[kOps], y[kOps];
#pragma unroll
    for (int r = 0; r < kWin; ++r) {
      x[r] = k_operand<kK>(kat[r], 1 - kb, r);
      if constexpr (kPv) y[r] = v_operand<kV>(vat[r >> 1], 1 - kb, r);
    }
    f32x16 next = {};
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int r = 0; r < kOps; ++r) {
      const int behind = kEach * (r + kWin <= kOps ? kWin - 1 : kOps - 1 - r);
      fa::lds_wait(x[r], behind + kEach - 1);
      next = F16::mfma(x[r], this->qreg[0][r], next);
#pragma unroll
      for (int i = 0; i < kPer; ++i) {
        const int it = r * kPer + i;
        st.pair(s[kb], kb, it / 4, it % 4, ref, pb_out, sum);
        if (it % 4 == 3) {
          st.add_group(sums, ref, kb * 2 + it / 4, sum);
          sum = 0.f;
        }
      }
      if constexpr (kPv) {
        fa::lds_wait(y[r], behind);
        st.acc[r >> 1] = F16::mfma(y[r], pb_in[r & 1], st.acc[r >> 1]);
      }
      if (r + kWin < kOps) {
        x[r + kWin] = k_operand<kK>(kat[r + kWin], 1 - kb, r + kWin);
        if constexpr (kPv) y[r + kWin] = v_operand<kV>(vat[(r + kWin) >> 1], 1 - kb, r + kWin);
      }
      __builtin_amdgcn_sched_barrier(0);
    }
    s[1 - kb] = next;
    return sums;
  }
  // The scores of half kb of a tile alone, and its values times the probabilities.
  __device__ __forceinline__ void scores(const uint8_t* k, int kb, f32x16& s) const {
    constexpr int kWin = 4;
    const uint32_t base = lds_addr(k);
    u32x4 x[kOps];
#pragma unroll
    for (int r = 0; r < kWin; ++r) x[r] = k_operand<0>(k_at(base, r), kb, r);
    s = f32x16{};
#pragma unroll
    for (int r = 0; r < kOps; ++r) {
      fa::lds_wait(x[r], r + kWin <= kOps ? kWin - 1 : kOps - 1 - r);
      s = F16::mfma(x[r], this->qreg[0][r], s);
      if (r + kWin < kOps) x[r + kWin] = k_operand<0>(k_at(base, r + kWin), kb, r + kWin);
    }
  }
  __device__ __forceinline__ void pv(const uint8_t* v, int kb, const u32x4 (&pb)[2]) {
    constexpr int kWin = 4;
    const uint32_t base = lds_addr(v);
    u32x4 y[kOps];
#pragma unroll
    for (int r = 0; r < kWin; ++r) y[r] = v_operand<0>(v_at(base, r), kb, r);
#pragma unroll
    for (int r = 0; r < kOps; ++r) {
      fa::lds_wait(y[r], 2 * (r + kWin <= kOps ? kWin - 1 : kOps - 1 - r));
      st.acc[r >> 1] = F16::mfma(y[r], pb[r & 1], st.acc[r >> 1]);
      if (r + kWin < kOps) y[r + kWin] = v_operand<0>(v_at(base, r + kWin), kb, r + kWin);
    }
  }
};

// The way of the tiles through a wave.  LDS has three stages for each of K and V, tile t in stage t % 3, which the clean steps know
// at compile time: operands lie at registers and constant offsets (478 us where each step adds them up).  In step j: the codes of
// K_{j+2} and V_{j+1}, asked for in the step before, go into stages that no wave reads any more, and those of K_{j+3}
// and V_{j+2} are asked for; then, half a tile (32 keys) at a time, the probabilities, between the products of the
// scores of the half behind and of the values of the half before.
struct WideAhead {
  u32x4 k, v;
  int n;             // number of tile j among the groups' current ones
  int c;             // j % 3
  u32x4 pb[2][2];    // probabilities of each half
};

// kStage: a.c, where tile j + 1 exists and all of the workgroup's rows attend all of tile j (whole: tiles of which they do); the second
// half's probabilities are left for the next step, whose kFirst is false, or for the caller.  -1: of any other tile.
template <int kStage, bool kFirst, int D, class E, class Q>
__device__ __forceinline__ void wide_step(WideState<D, E, Q>& w, const AttnArgs& p, int j, int end, int whole, uint8_t* ring, int most,
                                          int least, WideAhead& a, f32x16 (&s)[2]) {
  constexpr int T = WideState<D, E, Q>::T;
  Softmax<D>& st = w.st;
  constexpr bool kTail = kStage < 0;
  constexpr int kS1 = (kStage + 1) % 3, kS2 = (kStage + 2) % 3;
  const int c = kTail ? a.c : kStage;
  const int c1 = c == 2 ? 0 : c + 1, c2 = c == 0 ? 2 : c - 1;  // of j + 1, and of j + 2 and j - 1
  if (a.n == kBatch) {
    w.groups.advance(a.n);
    st.take_scales(w.groups.vs);
  }
  if (j + 2 < end) w.template store<false>(ring + c2 * T, w.kdst, a.k);
  if (j + 1 < end) {
    if (__is_same(Q, E4m3) && j + 1 >= whole) {
      w.template store<true>(ring + (3 + c1) * T, w.vdst, a.v);
    } else {
      w.template store<false>(ring + (3 + c1) * T, w.vdst, a.v);
    }
  }
  w.groups.ask(p, a.n, end * BKV);
  if (j + 2 < end) a.v = w.load(p.c.v, w.groups.template place<true>(a.n + 2, w.group), w.voff);
  if (j + 3 < end) a.k = w.load(p.c.k, w.groups.template place<false>(a.n + 3, w.group), w.koff);
  if constexpr (kTail) {
    if (j * BKV < most) {
      uint8_t *k_here = ring + c * T, *k_next = ring + c1 * T, *v_here = ring + (3 + c) * T;
      st.set_tile(w.groups.ks, a.n);
      w.scores(k_here, 1, s[1]);
      if ((j + 1) * BKV > least) st.hide(s, j, w.h);
      st.guard(s[0], 0, a.pb[0], st.probs(s[0], 0, a.pb[0]));
      w.pv(v_here, 0, a.pb[0]);
      st.guard(s[1], 1, a.pb[1], st.probs(s[1], 1, a.pb[1]));
      w.pv(v_here, 1, a.pb[1]);
      if ((j + 1) * BKV < most && j + 1 < end) w.scores(k_next, 0, s[0]);
    }
  } else {
    st.set_tile(w.groups.ks, a.n);
    st.guard(s[0], 0, a.pb[0], w.template half<0, !kFirst, kStage, kS2>(s, a.pb[1], a.pb[0]));
    st.guard(s[1], 1, a.pb[1], w.template half<1, true, kS1, kStage>(s, a.pb[0], a.pb[1]));
  }
  ++a.n;
  a.c = c1;
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  asm volatile("s_barrier" ::: "memory");
}

template <int D, class E, class Q>
__device__ __forceinline__ void wide_body(const AttnArgs& p) {
  using W = Wide<D>;
  constexpr int kWaves = W::kWaves, T = W::kTile, kThreads = kWaves * 64, kChunks = D / 8;
  constexpr bool kHasNan = __is_same(Q, E4m3);
  __shared__ __attribute__((aligned(256))) uint8_t ring[6 * T];

  kv::Share s = share_of(p);
  if (!s.live) return;
  s.row0 *= W::kRows;
  WideState<D, E, Q> w;
  const int tid = threadIdx.x;
  w.lane = tid & 63;
  w.wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  w.col = w.lane & 31;
  w.h = w.lane >> 5;
  w.init_tiles(p);
  w.groups.init(p, s, w.lane, 1);
  const int wave_row = s.row0 + w.wave * 32;
  const int query = load_query<D, false>(p, s, wave_row + w.col, w.h, w.qreg[0]);
  const Sequence seq(p, s.b);
  w.groups.len = seq.len;
  w.groups.poison = seq.bad;
  Softmax<D>& st = w.st;
  st.init();
  take_query<D, E>(p, seq, query, w.qreg[0], st.limit, st.power);
  int least = st.limit;
#pragma unroll
  for (int d = 1; d < 32; d *= 2) least = min(least, __shfl_xor(least, d, 64));
  least = __builtin_amdgcn_readfirstlane(least);
  const int most = wave_row < p.rows ? limit_of_rows(p, seq, wave_row, 32) : 0;

  const int total = (limit_of_rows(p, seq, s.row0, W::kRows) + BKV - 1) / BKV;
  const int per = p.per(total);
  const int begin = min(total, s.split * per), end = min(total, begin + per);
  w.found = 0;
  // tiles that all rows of the workgroup attend
  const int whole = min(end, least_of_rows(p, seq, s.row0, W::kRows) / BKV);
  if (begin < end) {
    WideAhead a;
    w.groups.start(p, begin, w.groups.entries(p, begin, seq.len));
    const auto load_k = [&](int i) { return w.load(p.c.k, w.groups.template place<false>(i, w.group), w.koff); };
    const auto load_v = [&](int i) { return w.load(p.c.v, w.groups.template place<true>(i, w.group), w.voff); };
    const int t1 = min(1, end - 1 - begin), t2 = min(2, end - 1 - begin);
    const u32x4 k0 = load_k(0), v0 = load_v(0), k1 = load_k(t1);
    a.k = load_k(t2);
    a.v = load_v(t1);
    st.take_scales(w.groups.vs);
    a.n = a.c = 0;  // tile begin in stage 0
    w.template store<false>(ring, w.kdst, k0);
    w.template store<false>(ring + T, w.kdst, k1);
    if (kHasNan && whole <= begin) {
      w.template store<true>(ring + 3 * T, w.vdst, v0);
    } else {
      w.template store<false>(ring + 3 * T, w.vdst, v0);
    }
    __syncthreads();
    w.init_places(ring);
    f32x16 s2[2];
    w.scores(ring, 0, s2[0]);
    int j = begin;
    const int clean = min(whole, end - 1);
    if (j < clean) {
      wide_step<0, true>(w, p, j, end, whole, ring, most, least, a, s2);
      for (++j; j + 2 < clean; j += 3) {
        wide_step<1, false>(w, p, j, end, whole, ring, most, least, a, s2);
        wide_step<2, false>(w, p, j + 1, end, whole, ring, most, least, a, s2);
        wide_step<0, false>(w, p, j + 2, end, whole, ring, most, least, a, s2);
      }
      w.pv(ring + 3 * T, 1, a.pb[1]);  // of stage 0
    }
    for (; j < end; ++j) wide_step<-1, false>(w, p, j, end, whole, ring, most, least, a, s2);
  }
  if (kHasNan && __syncthreads_or(w.found != 0) != 0) {
    for (int j = max(begin, whole); j < end; ++j) st.add_nan(p, s, j, w.h);
  }

  float l_run = st.l + other_half(st.l);
  if (w.groups.poison) l_run = __builtin_nanf("");
  const int written = written_of(p, s.b);
  if (p.splits > 1) {
    // the unnormalised part, from registers: lane (row, half h) holds d = 32 db + 8 rq + 4 h + 0..3
    const int row = wave_row + w.col;
    if (row < p.rows) {
      const int64_t place = static_cast<int64_t>(s.unit) * p.rows + row;
      if (w.h == 0) *reinterpret_cast<f32x4*>(p.part_ml + place * 4) = f32x4{st.m, l_run, st.M, 0.f};
#pragma unroll
      for (int db = 0; db < D / 32; ++db)
#pragma unroll
        for (int rq = 0; rq < 4; ++rq) {
          const f32x16& a = st.acc[db];
          *reinterpret_cast<f32x4*>(p.part_o + place * D + db * 32 + rq * 8 + w.h * 4) =
              f32x4{a[rq * 4], a[rq * 4 + 1], a[rq * 4 + 2], a[rq * 4 + 3]};
        }
    }
    return;
  }
  // rows of the block through the rings: 64 rows per stage
  const Result result(st.m, st.M, l_run);
  {
    const int brow = w.wave * 32 + w.col;
    uint8_t* os = ring + (brow >> 6) * T;
#pragma unroll
    for (int db = 0; db < D / 32; ++db)
#pragma unroll
      for (int rq = 0; rq < 4; ++rq) {
        const f32x16& a = st.acc[db];
        u32x2 x;
        x[0] = E::pack(result.of(a[rq * 4]), result.of(a[rq * 4 + 1]));
        x[1] = E::pack(result.of(a[rq * 4 + 2]), result.of(a[rq * 4 + 3]));
        *reinterpret_cast<u32x2*>(os + fa::k_off<D>(brow & 63, db * 4 + rq) + w.h * 8) = x;
      }
    int64_t o_at, lse_at;
    if (p.lse != nullptr && w.h == 0 && out_row(p, s, s.row0 + brow, written, o_at, lse_at)) {
      p.lse[lse_at] = kv::lse_of(st.m, l_run);
    }
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < W::kRows * kChunks / kThreads; ++i) {
    const int cc = tid + kThreads * i;
    const int row = cc / kChunks, ch = cc % kChunks;
    int64_t o_at, lse_at;
    if (!out_row(p, s, s.row0 + row, written, o_at, lse_at)) continue;
    *reinterpret_cast<u32x4*>(p.o + o_at + ch * 8) =
        *reinterpret_cast<const u32x4*>(ring + (row >> 6) * T + fa::k_off<D>(row & 63, ch));
  }
}

// Adds up the splits of a row, relative to the largest reference points.
template <int D, class E>
__device__ __forceinline__ void join_body(const AttnArgs& p) {
  const kv::JoinLanes<D> at(blockIdx.x, p.join_groups);
  const int64_t bh = at.row / p.rows;
  const int row = static_cast<int>(at.row - bh * p.rows);
  kv::Share s;
  s.b = static_cast<int>(bh / p.c.kv_heads);
  s.head = static_cast<int>(bh - static_cast<int64_t>(s.b) * p.c.kv_heads);
  if (s.b >= p.batch) return;
  const int written = written_of(p, s.b);
  int64_t o_at, lse_at;
  if (!out_row(p, s, row, written, o_at, lse_at)) return;  // all lanes of the row
  const int64_t first = static_cast<int64_t>(s.b) * p.splits * p.c.kv_heads + s.head;  // unit of split 0
  // each group of lanes its splits, against the largest so far, then the groups
  float m = -INFINITY, M = -INFINITY, l_run = 0.f, o[8] = {};
#pragma unroll 4
  for (int k = at.group; k < p.splits; k += at.groups) {
    const int64_t part = (first + static_cast<int64_t>(k) * p.c.kv_heads) * p.rows + row;
    const f32x4 ml = *reinterpret_cast<const f32x4*>(p.part_ml + part * 4);
    const f32x4 lo = *reinterpret_cast<const f32x4*>(p.part_o + part * D + at.ch * 8);
    const f32x4 hi = *reinterpret_cast<const f32x4*>(p.part_o + part * D + at.ch * 8 + 4);
    const auto weight = [](float x, float top) { return x == top ? 1.0f : __builtin_amdgcn_exp2f(x - top); };
    const float top = fmaxf(m, ml[0]), top_v = fmaxf(M, ml[2]);
    l_run = l_run * weight(m, top) + weight(ml[0], top) * ml[1];
    const float before = weight(M, top_v), f = weight(ml[2], top_v);
    m = top;
    M = top_v;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      o[e] = fmaf(f, lo[e], o[e] * before);
      o[4 + e] = fmaf(f, hi[e], o[4 + e] * before);
    }
  }
  const auto sum = [](float a, float b) { return a + b; };
  const auto most = [](float a, float b) { return fmaxf(a, b); };
  const float top = at.reduce(m, most), top_v = at.reduce(M, most);
  l_run = at.reduce(l_run * (m == top ? 1.0f : __builtin_amdgcn_exp2f(m - top)), sum);
  const float f = M == top_v ? 1.0f : __builtin_amdgcn_exp2f(M - top_v);
  m = top;
  M = top_v;
#pragma unroll
  for (int e = 0; e < 8; ++e) o[e] = at.reduce(o[e] * f, sum);
  if (at.group != 0) return;
  write_row<E>(p, s, row, at.ch, o, m, M, l_run, written);
}

}  // namespace c8
}  // namespace asc
