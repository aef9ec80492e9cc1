// Attention of query rows over the keys of a cache, with another number of keys than queries, shared
// key / value heads, per-sequence lengths, pages, and drafted tokens behind the cache: the device
// code of asc_cross_attention_fwd and asc_tree_attention.
//
// The queries that share a key / value head are its rows: row r is query r % n_q of the head's
// query head r / n_q.  A row's keys are the sequence's cached ones, all of them, and then the
// drafted ones that the tree mask names; o = sum_j p_j v_j / sum_j p_j with p_j = exp(s_j - m).
//
// The tile products, the probabilities and the moving reference point are FaState's.  What
// differs is where a tile's rows lie: lane l of a wave works out the place of the tile's key l (in
// units of 16 bytes: a page of the table and a row in it, or a row of the sequence), and each
// direct-to-LDS load takes the places of its rows from those lanes.  Rows past the last key come
// from a row of zeros, so nothing behind a sequence is read, whatever it holds.
//
// The probabilities (unnormalised, fp32 with their sums) are rounded to the element type for the product
// with the values, as matrix operands have to be: errors of 0.0023 of the results' norm in bf16 where one
// rounding of exact results leaves 0.0017 (0.00028 and 0.00021 in fp16).  A second product for what
// the rounding drops would add half to the matrix work.
//
//  - kv_wide: a workgroup owns up to 32 rows per wave and streams the keys once for all of them,
//    through rings of three LDS stages as fa_fwd_body.  The matrix units bound it, at the clock that
//    the board's power leaves: 4 x 32 heads, 4096 queries, 2048 keys, head_dim 128, bf16: 547 us,
//    1.0 PFLOP/s, matrix units busy 46%, at 1400 W of the board's 1400 and 2.0 GHz.  With shared heads and pages a chain of tiles and its
//    start and end do: 8 sequences of 1024 to 4096 keys, 64 drafted tokens, 32 / 8 heads: 47 us.
//  - kv_narrow: up to 32 rows; the workgroup's four waves take every fourth tile each.  HBM bounds it
//    over long caches: 8 sequences of up to 32768 keys in pages, 32 / 8 heads of 128, one token: 671 MB
//    in 117 us (5.7 TB/s); 16 sequences of up to 4096: 164 MB in 29.5 us (5.5).  Latency does over short
//    ones: 16 tokens, 500 keys: 10.8 us.
// Either way the keys may also be split over workgroups; kv_join adds the parts up (4.7 us for 512
// rows of 128 in 4 parts, 9 for 16384).
#pragma once

#include "flash_attn_kernels.h"

namespace asc {
namespace kv {

using fa::BKV;
using fa::f32x16;
using fa::FaState;
using fa::other_half;
using fa::u32x2;
using fa::u32x4;

typedef float f32x4 __attribute__((ext_vector_type(4)));

struct Strides {  // in units of 16 bytes
  uint32_t batch, head, seq;  // batch: of a page where there is a table
};

struct KvArgs {
  const uint16_t* q;
  uint16_t* o;
  float* lse;  // [batch, q_heads, n_q] or null
  int64_t q_batch, q_head, q_seq, o_batch, o_head, o_seq;  // elements
  const uint8_t* k;
  const uint8_t* v;
  const uint8_t* k_draft;  // null: no drafted keys
  const uint8_t* v_draft;
  Strides ks, vs, kds, vds;
  const int32_t* lengths;        // [batch] or null: capacity
  const int32_t* draft_lengths;  // [batch] or null: n_q
  const int32_t* table;          // [batch, table_stride] or null
  int64_t table_stride;
  const uint8_t* mask;  // [batch?, n_q, n_q] or null: a chain
  int64_t mask_batch, mask_row;
  int32_t mask_words;  // the mask's rows can be read four bytes at a time
  float* part_o;   // [unit][rows][D], unnormalised
  float* part_ml;  // [unit][rows][2]: reference point (log2), sum
  int32_t* infinite;  // [unit]: whether its drafted values hold infinities or NaN
  uint32_t num_pages, page_size, page_magic, page_shift;
  int32_t capacity;  // keys a sequence can have
  int32_t batch, kv_heads, group, n_q, rows, row_blocks;
  int32_t splits;  // of each sequence's keys
  int32_t join_groups;
  uint32_t units;  // batch * splits * kv_heads
  float scale_log2;
};

// Place of a tile's row that has no key, and the row read instead.
constexpr uint32_t kNone = 0xffffffffu;
static __device__ const u32x4 kZeroRow[16] = {};

// Cached keys of sequence b and its drafted ones; bad: a length outside what the call can hold.
__device__ __forceinline__ int clamped(int n, int most, bool& bad) {
  bad = bad || n < 0 || n > most;
  return n < 0 ? 0 : (n > most ? most : n);
}
template <bool kTree>
__device__ __forceinline__ void keys_of(const KvArgs& p, int b, int& len, int& drafts, bool& bad) {
  len = clamped(p.lengths ? p.lengths[b] : p.capacity, p.capacity, bad);
  drafts = 0;
  if constexpr (kTree) drafts = clamped(p.draft_lengths ? p.draft_lengths[b] : p.n_q, p.n_q, bad);
}

// One workgroup's share: a sequence's key / value head, a block of its rows, a split of its keys;
// `unit` is where its part goes.
struct Share {
  int b, head, row0, split;
  uint32_t unit;
  bool live;
};

// Workgroup i runs on XCD i % 8.  The row blocks of one range of keys run on one XCD one after the
// other: they read the same keys through its L2.
//
// A sequence's keys may be split over workgroups, each with an even share of its tiles.
__device__ __forceinline__ Share share_of(const KvArgs& p) {
  const uint32_t slot = blockIdx.x >> 3;
  const uint32_t per = slot / p.row_blocks;
  Share s;
  s.unit = per * 8 + (blockIdx.x & 7);
  s.live = s.unit < p.units;
  s.row0 = static_cast<int>(slot - per * p.row_blocks);
  const uint32_t range = s.unit / p.kv_heads;
  s.head = static_cast<int>(s.unit - range * p.kv_heads);
  s.b = static_cast<int>(range / p.splits);
  s.split = static_cast<int>(range - static_cast<uint32_t>(s.b) * p.splits);
  return s;
}

// kTree: there may be a table of pages, drafted keys and a mask over them.
template <int D, int kWaves, class E, bool kTree>
struct KvState : FaState<D, kWaves, 1, E, kTree> {
  using Base = FaState<D, kWaves, 1, E, kTree>;
  using Base::col;
  using Base::h;
  using Base::kKSteps;
  using Base::kLoadsPerWave;
  using Base::kRowsPerLoad;
  using Base::kTileBytes;
  using Base::lane;
  using Base::wave;

  int len, drafts;     // cached and drafted keys of the sequence
  int cached;          // tiles of cached keys; the drafted ones follow in tiles of their own
  int query;           // this lane's query (of n_q), or -1: no row
  const int32_t* table;
  int* infinite;       // LDS, one of each wave: 1 where it has loaded infinite or NaN drafted values
  int wave_of;         // in the workgroup
  uint8_t* ids;        // LDS, 256 bytes of this wave: the fetched entries of a tile's keys
  uint32_t drafted;    // mask_bits of the first drafted tile
  uint32_t k0, v0, kd0, vd0;  // the sequence's first row (16-byte units)
  uint32_t k_step, v_step;    // from row to row
  bool even;                  // whole tiles lie in one piece, within 2 GiB of it
  const uint8_t* mask;
  bool poison;         // a page or a length outside the cache: the rows' results are NaN

  __device__ __forceinline__ void init(const KvArgs& p, const Share& s) {
    poison = false;
    keys_of<kTree>(p, s.b, len, drafts, poison);
    if (kTree) infinite[wave_of] = 0;
    cached = (len + BKV - 1) / BKV;
    const bool paged = kTree && p.table != nullptr;
    k0 = s.head * p.ks.head + (paged ? 0 : s.b * p.ks.batch);
    v0 = s.head * p.vs.head + (paged ? 0 : s.b * p.vs.batch);
    k_step = p.ks.seq;
    v_step = p.vs.seq;
    even = (!paged || p.page_size % BKV == 0) && max(k_step, v_step) < (1u << 31) / (16 * BKV);
    if constexpr (kTree) {
      table = paged ? p.table + s.b * p.table_stride : nullptr;
      kd0 = s.head * p.kds.head + s.b * p.kds.batch;
      vd0 = s.head * p.vds.head + s.b * p.vds.batch;
      mask = p.mask ? p.mask + s.b * p.mask_batch : nullptr;
      drafted = 0;
    }

    constexpr int kLanesPerRow = 64 / kRowsPerLoad;
    const int rr = lane / kLanesPerRow, pos = lane % kLanesPerRow;
#pragma unroll
    for (int i = 0; i < Base::kKOffs; ++i) {
      const int row = kRowsPerLoad * ((wave * kLoadsPerWave + i) & 3) + rr;
      this->voff_k[i] = (pos ^ fa::kswz<D>(row)) << 4;
    }
    this->voff_v = (pos ^ fa::vswz<D>(rr)) << 4;
    constexpr int kK = kTree ? 1 : kKSteps, kV = kTree ? 1 : Base::kDBlocks;
#pragma unroll
    for (int kk = 0; kk < kK; ++kk) this->kaddr[kk] = fa::k_off<D>(col, kk * 2 + h);
    const int g_lane = lane & 15;
    const int tr_col = ((lane >> 4) & 1) * 16 + (g_lane & 3) * 4;
#pragma unroll
    for (int db = 0; db < kV; ++db) this->vaddr[db] = fa::v_off<D>(h * 4 + (g_lane >> 2), db * 32 + tr_col);
  }

  __device__ __forceinline__ int tiles() const { return cached + (drafts + BKV - 1) / BKV; }

  // Address of the table entry of tile j's key of this lane (of the last key behind it), j < cached.
  __device__ __forceinline__ const int32_t* entry(const KvArgs& p, int j) const {
    const int key = min(j * BKV + lane, len - 1);
    // key / page_size: the magic's error, below page_size, times key stays under 2^(31 + shift)
    return table + static_cast<uint32_t>((static_cast<uint64_t>(key) * p.page_magic) >> (31 + p.page_shift));
  }
  __device__ __forceinline__ uint32_t entry_now(const KvArgs& p, int j) const {
    if (!kTree || table == nullptr || j >= cached) return 0;
    return static_cast<uint32_t>(*entry(p, j));
  }
  // Asks for tile j's entries, a tile ahead of their use, straight into LDS: a load to registers
  // would be waited for with all loads of tiles behind it, as the compiler cannot count those
  // past a branch.  Sent before a step's tiles, the step's own wait covers it.
  __device__ __forceinline__ void fetch(const KvArgs& p, int j) const {
    if (!kTree || table == nullptr || j >= cached) return;
    __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)entry(p, j),
                                     (__attribute__((address_space(3))) void*)ids, 4, 0, 0);
  }
  __device__ __forceinline__ uint32_t fetched(int j) const {
    if (!kTree || table == nullptr || j >= cached) return 0;
    uint32_t r;
    asm volatile("ds_read_b32 %0, %1\n\ts_waitcnt lgkmcnt(0)" : "=v"(r) : "v"(fa::lds_addr(ids) + lane * 4) : "memory");
    return r;
  }

  // Places of tile j's keys, one per lane, of its table entry.
  __device__ __forceinline__ void places(const KvArgs& p, int j, uint32_t id, uint32_t& ik, uint32_t& iv) {
    const int key = (j < cached ? j : j - cached) * BKV + lane;
    if (!kTree || j < cached) {
      if (kTree && table != nullptr) {
        const uint32_t at = min(key, len - 1);
        const uint32_t page = static_cast<uint32_t>((static_cast<uint64_t>(at) * p.page_magic) >> (31 + p.page_shift));
        const uint32_t row = at - page * p.page_size;
        const bool bad = id >= p.num_pages;
        poison = poison || __builtin_amdgcn_ballot_w64(bad) != 0;
        if (bad) id = 0;
        ik = k0 + id * p.ks.batch + row * p.ks.seq;
        iv = v0 + id * p.vs.batch + row * p.vs.seq;
      } else {
        ik = k0 + key * p.ks.seq;
        iv = v0 + key * p.vs.seq;
      }
      if (key >= len) ik = iv = kNone;
    } else {
      ik = key < drafts ? kd0 + key * p.kds.seq : kNone;
      iv = key < drafts ? vd0 + key * p.vds.seq : kNone;
    }
  }

  // Tile j of K (kIsV false) or V, whose rows' places the lanes hold, into one LDS stage.
  template <bool kIsV>
  __device__ __forceinline__ void load(const KvArgs& p, uint8_t* dst, int j, uint32_t places) const {
    uint64_t base = reinterpret_cast<uint64_t>(kIsV ? p.v : p.k);
    if constexpr (kTree) {
      uint64_t draft = reinterpret_cast<uint64_t>(kIsV ? p.v_draft : p.k_draft);
      asm("" : "+s"(base), "+s"(draft));  // selected in registers, not from a table in scratch memory
      if (j >= cached) base = draft;
    }
    const bool whole = (j + 1) * BKV <= len;
    int wave_lds = wave * (kLoadsPerWave * 1024);
    asm volatile("" : "+s"(wave_lds));
    constexpr int kLanesPerRow = 64 / kRowsPerLoad;
    const int rr = lane / kLanesPerRow;
    if (whole && even) {
      // rows at a fixed distance from the tile's first: one scalar base and an offset per lane
      const uint32_t first = __builtin_amdgcn_readfirstlane(places);
      base += static_cast<uint64_t>(first) * 16;
      const uint32_t stride = (kIsV ? v_step : k_step) * 16;
#pragma unroll
      for (int i = 0; i < kLoadsPerWave; ++i) {
        const uint32_t row = kRowsPerLoad * (wave * kLoadsPerWave + i);
        const uint32_t off = rr * stride + (kIsV ? this->voff_v : this->voff_k[i & 3]);
        __builtin_amdgcn_global_load_lds(
            (const __attribute__((address_space(1))) void*)(reinterpret_cast<const uint8_t*>(base + row * stride) + off),
            (__attribute__((address_space(3))) void*)(dst + wave_lds + i * 1024), 16, 0, 0);
      }
      return;
    }
    if (kTree && kIsV && j >= cached) {
      load_drafted_values(base, dst + wave_lds, places);
      return;
    }
#pragma unroll
    for (int i = 0; i < kLoadsPerWave; ++i) {
      const int row = kRowsPerLoad * (wave * kLoadsPerWave + i) + rr;
      const uint32_t at =
          static_cast<uint32_t>(__builtin_amdgcn_ds_bpermute(row * 4, static_cast<int>(places)));
      const uint8_t* src = reinterpret_cast<const uint8_t*>(base + static_cast<uint64_t>(at) * 16);
      if (!whole) src = at == kNone ? reinterpret_cast<const uint8_t*>(kZeroRow) : src;
      __builtin_amdgcn_global_load_lds(
          (const __attribute__((address_space(1))) void*)(src + (kIsV ? this->voff_v : this->voff_k[i & 3])),
          (__attribute__((address_space(3))) void*)(dst + wave_lds + i * 1024), 16, 0, 0);
    }
  }

  // Drafted values go through registers: infinities and NaN become zeros, because 0 times those is
  // not 0 and a row must not see the values of a token that it does not attend.  The rows that
  // attend it get them back at the end (add_infinite).
  __device__ __forceinline__ void load_drafted_values(uint64_t base, uint8_t* dst, uint32_t places) const {
    constexpr uint32_t kExp = __is_same(E, fa::Bf16) ? 0x7f80u : 0x7c00u;
    const int rr = lane / (64 / kRowsPerLoad);
    bool found = false;
#pragma unroll 4
    for (int i = 0; i < kLoadsPerWave; ++i) {
      const int row = kRowsPerLoad * (wave * kLoadsPerWave + i) + rr;
      const uint32_t at =
          static_cast<uint32_t>(__builtin_amdgcn_ds_bpermute(row * 4, static_cast<int>(places)));
      u32x4 w = {0, 0, 0, 0};
      if (at != kNone) w = *reinterpret_cast<const u32x4*>(base + static_cast<uint64_t>(at) * 16 + this->voff_v);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const bool low = (w[e] & kExp) == kExp, high = (w[e] >> 16 & kExp) == kExp;
        found = found || low || high;
        w[e] &= (low ? 0xffff0000u : ~0u) & (high ? 0xffffu : ~0u);
      }
      *reinterpret_cast<u32x4*>(dst + i * 1024 + lane * 16) = w;
    }
    if (__builtin_amdgcn_ballot_w64(found) != 0) infinite[wave_of] = 1;
  }

  __device__ __forceinline__ bool needs_mask(int j) const { return (j + 1) * BKV > len; }

  // Scores of tile j: -inf for keys that the lane's row does not attend.
  __device__ __forceinline__ void hide(const KvArgs& p, f32x16 (&s)[1][2], int j) const {
    if (!kTree || j < cached) {
#pragma unroll
      for (int kb = 0; kb < 2; ++kb)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          if (j * BKV + kb * 32 + (r >> 2) * 8 + h * 4 + (r & 3) >= len) s[0][kb][r] = -INFINITY;
        }
      return;
    }
    uint32_t seen = drafted;
    if (j > cached) {
      uint32_t words[8];
      mask_words(p, (j - cached) * BKV, words);
      seen = mask_bits((j - cached) * BKV, words);
    }
#pragma unroll
    for (int kb = 0; kb < 2; ++kb)
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        if (!((seen >> (kb * 16 + r)) & 1)) s[0][kb][r] = -INFINITY;
      }
  }

  // Which of the drafted keys first .. first + 63 this lane's row attends: bit 16 kb + r for score
  // register r of block kb, keys 32 kb + 8 (r / 4) + 4 h + r % 4, so four bytes of the mask's row
  // each.  The words are asked for ahead of the tiles.
  __device__ __forceinline__ void mask_words(const KvArgs& p, int first, uint32_t (&words)[8]) const {
    if (mask == nullptr) return;
    const uint8_t* row = mask + static_cast<int64_t>(query < 0 ? 0 : query) * p.mask_row;
    if (p.mask_words) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int key = first + (i >> 2) * 32 + (i & 3) * 8 + h * 4;
        words[i] = *reinterpret_cast<const uint32_t*>(row + min(key, p.n_q - 4));
      }
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        words[i] = 0;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int key = first + (i >> 2) * 32 + (i & 3) * 8 + h * 4 + e;
          words[i] |= static_cast<uint32_t>(row[min(key, p.n_q - 1)]) << (8 * e);
        }
      }
    }
  }
  __device__ __forceinline__ uint32_t mask_bits(int first, const uint32_t (&words)[8]) const {
    uint32_t seen = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int key = first + (i >> 2) * 32 + (i & 3) * 8 + h * 4;
      uint32_t w = words[i];  // four flags in the lowest bits of its bytes, then next to each other
      w = (w | w >> 4) & 0x0f0f0f0fu;
      w = (w | w >> 2) & 0x03030303u;
      w = (w | w >> 1) & 0x01010101u;
      w = w * 0x10204080u >> 28;
      if (mask == nullptr) w = (1u << min(max(query + 1 - key, 0), 4)) - 1;  // a chain: keys <= query
      const int left = query < 0 ? 0 : min(max(drafts - key, 0), 4);
      seen |= (w & ((1u << left) - 1)) << (4 * i);
    }
    return seen;
  }

  // Whether the reference point has to move: a lane's sum of probabilities is too large, or a row
  // has had no key yet and so no reference point.
  __device__ __forceinline__ bool out_of_range(float sum) const {
    return __builtin_amdgcn_ballot_w64(sum > E::kTileSumLimit || this->m_run[0] == -INFINITY) != 0;
  }

  // This lane's row of the block: its query and where its output and statistics lie.
  __device__ __forceinline__ void set_query(const KvArgs& p, const Share& s, int row, int64_t& q_at) {
    query = -1;
    q_at = 0;
    if (row < p.rows) {
      const int g = row / p.n_q;
      query = row - g * p.n_q;
      q_at = s.b * p.q_batch + static_cast<int64_t>(s.head * p.group + g) * p.q_head + query * p.q_seq;
    }
  }

  __device__ __forceinline__ void load_query(const KvArgs& p, int64_t q_at) {
#pragma unroll
    for (int ks = 0; ks < kKSteps; ++ks) {
      this->qreg[0][ks] = u32x4{0, 0, 0, 0};
      if (query >= 0) this->qreg[0][ks] = *reinterpret_cast<const u32x4*>(p.q + q_at + ks * 16 + h * 8);
    }
#pragma unroll
    for (int i = 0; i < Base::kDBlocks; ++i) this->acc_o[0][i] = f32x16{};
    this->m_run[0] = -INFINITY;
    this->l_part[0] = 0.f;
    this->scale_log2 = p.scale_log2;
  }
};

// Output row `row` of the share: its query and head, false where nothing is written.
__device__ __forceinline__ bool out_row(const KvArgs& p, const Share& s, int row, int written, int64_t& o_at,
                                        int64_t& lse_at) {
  if (row >= p.rows) return false;
  const int g = row / p.n_q, query = row - g * p.n_q;
  if (query >= written) return false;
  const int64_t head = s.head * p.group + g;
  o_at = s.b * p.o_batch + head * p.o_head + query * p.o_seq;
  lse_at = (static_cast<int64_t>(s.b) * p.kv_heads * p.group + head) * p.n_q + query;
  return true;
}

// Queries of sequence b that are written: those behind its drafted tokens are left as they were (all, where
// their number is negative; one above n_q leaves none, and they are NaN).
__device__ __forceinline__ int written_of(const KvArgs& p, int b) {
  return p.k_draft && p.draft_lengths ? p.draft_lengths[b] : p.n_q;
}

// 0 for a row without keys; NaN stays NaN.
__device__ __forceinline__ float inverse_sum(float l) { return l == 0.f ? 0.f : 1.0f / l; }

__device__ __forceinline__ float lse_of(float m, float l) { return (m + __log2f(l)) * 0.69314718055994530942f; }

template <class E>
__device__ __forceinline__ u32x4 pack8(const float (&o)[8], float scale) {
  u32x4 w;
#pragma unroll
  for (int e = 0; e < 4; ++e) w[e] = E::pack(o[2 * e] * scale, o[2 * e + 1] * scale);
  return w;
}
template <class E>
__device__ __forceinline__ void unpack(const u32x4& w, float (&o)[8]) {
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const uint16_t bits = static_cast<uint16_t>(w[e / 2] >> (e % 2 * 16));
    o[e] = __is_same(E, fa::Bf16) ? bf16_to_f32(bits) : f16_to_f32(bits);
  }
}

// What the infinities and NaN among the drafted values that a row attends add to eight of its
// results: rare, so one key after the other.
template <class E>
__device__ __forceinline__ void add_infinite(const KvArgs& p, int b, int head, int query, int ch, float (&o)[8]) {
  typedef uint16_t u16x8 __attribute__((ext_vector_type(8)));
  bool bad = false;
  const int drafts = clamped(p.draft_lengths ? p.draft_lengths[b] : p.n_q, p.n_q, bad);
  const uint8_t* mask = p.mask ? p.mask + b * p.mask_batch + query * p.mask_row : nullptr;
  const uint8_t* v = p.v_draft + (static_cast<uint64_t>(b) * p.vds.batch + static_cast<uint64_t>(head) * p.vds.head) * 16;
  for (int key = 0; key < drafts; ++key) {
    if (!(mask ? mask[key] != 0 : key <= query)) continue;
    const u16x8 x = *reinterpret_cast<const u16x8*>(v + static_cast<uint64_t>(key) * p.vds.seq * 16 + ch * 16);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float f = __is_same(E, fa::Bf16) ? bf16_to_f32(x[e]) : f16_to_f32(x[e]);
      if (!(fabsf(f) < INFINITY)) o[e] += f;
    }
  }
}

// One pipeline step for tile j of [.., end), as fa_step: on entry LDS holds K_{j+1} and V_j, sc the
// masked scores of tile j.  iv2: places of V_{j+2}; the table entries of tile j+3 have been fetched.
// kTail false: tile j+1 exists and is whole, and its scores are taken into sn between the
// probabilities of tile j.  kTail true: any tile, one thing after the other, the next scores into sc.
template <bool kTail, class St>
__device__ __forceinline__ void kv_step(St& st, const KvArgs& p, int j, int end, uint8_t* ring, int c, bool act,
                                        uint32_t& iv2, f32x16 (&sc)[1][2], f32x16 (&sn)[1][2]) {
  constexpr int T = St::kTileBytes;
  constexpr int L = St::kLoadsPerWave;
  const int c1 = c == 2 ? 0 : c + 1;
  const int c2 = c == 0 ? 2 : c - 1;
  const bool load_v = j + 2 < end, load_k = j + 3 < end;
  uint32_t ik3 = 0, iv3 = 0;
  if (load_k) {
    st.places(p, j + 3, st.fetched(j + 3), ik3, iv3);
    st.fetch(p, j + 4);
  }
  if (load_v) st.template load<true>(p, ring + (3 + c2) * T, j + 2, iv2);
  if (load_k) st.template load<false>(p, ring + c * T, j + 3, ik3);
  iv2 = iv3;
  if (!kTail || act) {
    u32x4 pb[1][2][2];
    float rs[1];
    if constexpr (kTail) {
      rs[0] = st.probs(0, sc[0], pb[0]);
    } else {
      st.scores_probs(ring + c1 * T, sn, sc, pb, rs);
    }
    if (st.out_of_range(rs[0])) {
      st.raise(0, st.tile_max(sc[0]));
      rs[0] = st.probs(0, sc[0], pb[0]);
    }
    st.l_part[0] += rs[0];
    st.pv(ring + (3 + c) * T, pb);
    if constexpr (kTail) {
      if (j + 1 < end) {
        st.scores(ring + c1 * T, sc);
        if (st.needs_mask(j + 1)) st.hide(p, sc, j + 1);
      }
    }
  }
  if (load_k) {
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(2 * L) : "memory");
  } else if (load_v) {
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(L) : "memory");
  } else {
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
  }
  asm volatile("s_barrier" ::: "memory");
}

template <int D>
struct Wide {
  static constexpr int kWaves = D == 128 ? 8 : 4, kWgPerCu = D == 128 ? 1 : 2;
  static constexpr int kRows = 32 * kWaves;
};

template <int D, class E, bool kTree>
__device__ __forceinline__ void kv_wide_body(const KvArgs& p) {
  constexpr int kWaves = Wide<D>::kWaves;
  using St = KvState<D, kWaves, E, kTree>;
  constexpr int T = St::kTileBytes;
  constexpr int L = St::kLoadsPerWave;
  constexpr int kThreads = kWaves * 64;
  constexpr int kChunks = D / 8;
  __shared__ __attribute__((aligned(256))) uint8_t ring[6 * T];
  __shared__ __attribute__((aligned(16))) uint8_t ids[kTree ? kWaves * 256 : 16];
  __shared__ int infinite[kWaves];

  Share s = share_of(p);
  if (!s.live) return;
  s.row0 *= Wide<D>::kRows;
  St st;
  const int tid = threadIdx.x;
  if (kWaves == 8 && (tid >> 6) < 4) __builtin_amdgcn_s_setprio(1);
  st.lane = tid & 63;
  st.wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  st.col = st.lane & 31;
  st.h = st.lane >> 5;
  st.ids = ids + (kTree ? st.wave * 256 : 0);
  st.infinite = infinite;
  st.wave_of = st.wave;
  st.init(p, s);
  const int wave_row = s.row0 + st.wave * 32;
  const bool act = wave_row < p.rows;
  int64_t q_at;
  st.set_query(p, s, wave_row + st.col, q_at);
  st.load_query(p, q_at);

  const int total = st.tiles();
  const int per = (total + p.splits - 1) / p.splits;
  const int begin = min(total, s.split * per), end = min(total, begin + per);
  if (begin < end) {
    uint32_t ik0, ik1 = 0, ik2 = 0, iv0, iv1 = 0, iv2 = 0;
    // the mask's words are asked for with the table's entries, ahead of the tiles
    const bool drafted = kTree && begin <= st.cached && st.cached < end;
    uint32_t words[8] = {};
    if (drafted) st.mask_words(p, 0, words);
    {
      const uint32_t id0 = st.entry_now(p, begin);
      const uint32_t id1 = begin + 1 < end ? st.entry_now(p, begin + 1) : 0;
      const uint32_t id2 = begin + 2 < end ? st.entry_now(p, begin + 2) : 0;
      st.places(p, begin, id0, ik0, iv0);
      if (begin + 1 < end) st.places(p, begin + 1, id1, ik1, iv1);
      if (begin + 2 < end) st.places(p, begin + 2, id2, ik2, iv2);
    }
    if (begin + 3 < end) st.fetch(p, begin + 3);
    st.template load<false>(p, ring, begin, ik0);
    st.template load<true>(p, ring + 3 * T, begin, iv0);
    if (begin + 1 < end) {
      st.template load<false>(p, ring + T, begin + 1, ik1);
      st.template load<true>(p, ring + 4 * T, begin + 1, iv1);
    }
    if (begin + 2 < end) st.template load<false>(p, ring + 2 * T, begin + 2, ik2);
    if (drafted) st.drafted = st.mask_bits(0, words);
    if (begin + 2 < end) {
      asm volatile("s_waitcnt vmcnt(%0)" ::"n"(2 * L) : "memory");
    } else if (begin + 1 < end) {
      asm volatile("s_waitcnt vmcnt(%0)" ::"n"(L) : "memory");
    } else {
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    }
    asm volatile("s_barrier" ::: "memory");
    f32x16 sa[1][2], sb[1][2];
    st.scores(ring, sa);
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    asm volatile("s_barrier" ::: "memory");
    if (st.needs_mask(begin)) st.hide(p, sa, begin);
    if (act) st.m_run[0] = st.tile_max(sa[0]);  // nothing to rescale yet
    int j = begin, c = 0;
    if (act) {
      const int whole = min(end, st.len / BKV);
      for (; j + 2 < whole; j += 2) {
        kv_step<false>(st, p, j, end, ring, c, true, iv2, sa, sb);
        c = c == 2 ? 0 : c + 1;
        kv_step<false>(st, p, j + 1, end, ring, c, true, iv2, sb, sa);
        c = c == 2 ? 0 : c + 1;
      }
    }
    for (; j < end; ++j) {
      kv_step<true>(st, p, j, end, ring, c, act, iv2, sa, sa);
      c = c == 2 ? 0 : c + 1;
    }
  }

  float l_run = st.l_part[0] + other_half(st.l_part[0]);
  if (st.poison) l_run = __builtin_nanf("");
  const int written = written_of(p, s.b);
  const auto any_infinite = [&] {
    int any = 0;
    for (int w = 0; w < kWaves; ++w) any |= infinite[w];
    return any;
  };
  if (p.splits > 1) {
    if constexpr (kTree) {
      __syncthreads();
      if (tid == 0) p.infinite[s.unit] = any_infinite();
    }
    // the unnormalised part, from registers: lane (row, half h) holds d = 32 db + 8 rq + 4 h + 0..3
    const int row = wave_row + st.col;
    if (row < p.rows) {
      const int64_t at = static_cast<int64_t>(s.unit) * p.rows + row;
      if (st.h == 0) *reinterpret_cast<float2*>(p.part_ml + at * 2) = make_float2(st.m_run[0], l_run);
      if (begin < end) {
#pragma unroll
        for (int db = 0; db < St::kDBlocks; ++db)
#pragma unroll
          for (int rq = 0; rq < 4; ++rq) {
            const f32x16& a = st.acc_o[0][db];
            *reinterpret_cast<f32x4*>(p.part_o + at * D + db * 32 + rq * 8 + st.h * 4) =
                f32x4{a[rq * 4], a[rq * 4 + 1], a[rq * 4 + 2], a[rq * 4 + 3]};
          }
      }
    }
    return;
  }
  // rows of the block through the rings (no load is in flight): 64 rows per stage
  const float inv = inverse_sum(l_run);
  {
    const int brow = st.wave * 32 + st.col;
    uint8_t* os = ring + (brow >> 6) * T;
#pragma unroll
    for (int db = 0; db < St::kDBlocks; ++db)
#pragma unroll
      for (int rq = 0; rq < 4; ++rq) {
        const f32x16& a = st.acc_o[0][db];
        u32x2 w;
        w[0] = E::pack(a[rq * 4] * inv, a[rq * 4 + 1] * inv);
        w[1] = E::pack(a[rq * 4 + 2] * inv, a[rq * 4 + 3] * inv);
        *reinterpret_cast<u32x2*>(os + fa::k_off<D>(brow & 63, db * 4 + rq) + st.h * 8) = w;
      }
    int64_t o_at, lse_at;
    if (p.lse != nullptr && st.h == 0 && out_row(p, s, s.row0 + brow, written, o_at, lse_at)) {
      p.lse[lse_at] = lse_of(st.m_run[0], l_run);
    }
  }
  __syncthreads();
  const bool add = kTree && any_infinite();
#pragma unroll
  for (int i = 0; i < Wide<D>::kRows * kChunks / kThreads; ++i) {
    const int cc = tid + kThreads * i;
    const int row = cc / kChunks, ch = cc % kChunks;
    int64_t o_at, lse_at;
    if (!out_row(p, s, s.row0 + row, written, o_at, lse_at)) continue;
    u32x4 w = *reinterpret_cast<const u32x4*>(ring + (row >> 6) * T + fa::k_off<D>(row & 63, ch));
    if (add) {
      float o[8];
      unpack<E>(w, o);
      add_infinite<E>(p, s.b, s.head, (s.row0 + row) % p.n_q, ch, o);
      w = pack8<E>(o, 1.0f);
    }
    *reinterpret_cast<u32x4*>(p.o + o_at + ch * 8) = w;
  }
}

template <int D>
struct Narrow {
  static constexpr int kWaves = 4, kWgPerCu = D == 64 ? 2 : 1;
  static constexpr int kRows = 32;
};

template <int D, class E, bool kTree>
__device__ __forceinline__ void kv_narrow_body(const KvArgs& p) {
  using St = KvState<D, 1, E, kTree>;
  constexpr int kWaves = Narrow<D>::kWaves;
  constexpr int T = St::kTileBytes;
  constexpr int L = St::kLoadsPerWave;
  constexpr int kRow = D * 4;
  static_assert(Narrow<D>::kRows * kRow <= 2 * T, "a wave's part reuses its tiles");
  __shared__ __attribute__((aligned(256))) uint8_t lds[kWaves * 2 * T];
  __shared__ float stats[2][kWaves][Narrow<D>::kRows];
  __shared__ __attribute__((aligned(16))) uint8_t ids[kTree ? kWaves * 256 : 16];
  __shared__ int infinite[kWaves];

  Share s = share_of(p);
  if (!s.live) return;
  s.row0 *= Narrow<D>::kRows;
  St st;
  const int tid = threadIdx.x;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  uint8_t* kring = lds + wave * 2 * T;
  uint8_t* vring = kring + T;
  st.lane = tid & 63;
  st.wave = 0;
  st.col = st.lane & 31;
  st.h = st.lane >> 5;
  st.ids = ids + (kTree ? wave * 256 : 0);
  st.infinite = infinite;
  st.wave_of = wave;
  st.init(p, s);
  int64_t q_at;
  st.set_query(p, s, s.row0 + st.col, q_at);
  st.load_query(p, q_at);

  const int total = st.tiles();
  const int per = (total + p.splits - 1) / p.splits;
  const int begin = min(total, s.split * per), end = min(total, begin + per);
  uint32_t ik = 0, iv = 0, iv_next = 0;
  if (begin + wave < end) {
    const bool drafted =
        kTree && st.cached >= begin + wave && st.cached < end && (st.cached - begin - wave) % kWaves == 0;
    uint32_t words[8] = {};
    if (drafted) st.mask_words(p, 0, words);
    st.places(p, begin + wave, st.entry_now(p, begin + wave), ik, iv);
    if (begin + wave + kWaves < end) st.fetch(p, begin + wave + kWaves);
    st.template load<false>(p, kring, begin + wave, ik);
    st.template load<true>(p, vring, begin + wave, iv);
    if (drafted) st.drafted = st.mask_bits(0, words);
  }
  for (int j = begin + wave; j < end; j += kWaves) {
    const bool next = j + kWaves < end;
    // all but V_j have landed
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"(L) : "memory");
    f32x16 sc[1][2];
    st.scores(kring, sc);
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    if (next) {
      st.places(p, j + kWaves, st.fetched(j + kWaves), ik, iv_next);
      st.template load<false>(p, kring, j + kWaves, ik);
    }
    if (st.needs_mask(j)) st.hide(p, sc, j);
    if (j == begin + wave) st.m_run[0] = st.tile_max(sc[0]);  // nothing to rescale yet
    u32x4 pb[1][2][2];
    float rs = st.probs(0, sc[0], pb[0]);
    if (st.out_of_range(rs)) {
      st.raise(0, st.tile_max(sc[0]));
      rs = st.probs(0, sc[0], pb[0]);
    }
    st.l_part[0] += rs;
    if (next) {
      asm volatile("s_waitcnt vmcnt(%0)" ::"n"(L) : "memory");  // all but K of the next tile
    } else {
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    }
    st.pv(vring, pb);
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    if (next) {
      if (j + 2 * kWaves < end) st.fetch(p, j + 2 * kWaves);
      st.template load<true>(p, vring, j + kWaves, iv_next);
    }
  }

  // the waves' parts, relative to their own reference points, through LDS
  const auto part_off = [](int row, int c) { return row * kRow + ((c ^ (row & 15)) << 4); };
  {
    float l = st.l_part[0] + other_half(st.l_part[0]);
    if (st.poison) l = __builtin_nanf("");
    if (st.h == 0) {
      stats[0][wave][st.col] = st.m_run[0];
      stats[1][wave][st.col] = l;
    }
#pragma unroll
    for (int db = 0; db < St::kDBlocks; ++db)
#pragma unroll
      for (int rq = 0; rq < 4; ++rq) {
        const f32x16& a = st.acc_o[0][db];
        *reinterpret_cast<f32x4*>(kring + part_off(st.col, db * 8 + rq * 2 + st.h)) =
            f32x4{a[rq * 4], a[rq * 4 + 1], a[rq * 4 + 2], a[rq * 4 + 3]};
      }
  }
  __syncthreads();
  const int written = written_of(p, s.b);
  int add = 0;
  if constexpr (kTree) {
    for (int w = 0; w < kWaves; ++w) add |= infinite[w];
    if (p.splits > 1 && tid == 0) p.infinite[s.unit] = add;
  }
#pragma unroll
  for (int i = 0; i < Narrow<D>::kRows * (D / 8) / (kWaves * 64); ++i) {
    const int cc = tid + kWaves * 64 * i;
    const int row = cc / (D / 8), ch = cc % (D / 8);
    if (s.row0 + row >= p.rows) continue;
    float m = stats[0][0][row];
#pragma unroll
    for (int w = 1; w < kWaves; ++w) m = fmaxf(m, stats[0][w][row]);
    float f[kWaves], l_run = 0.f;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      const float mw = stats[0][w][row];
      f[w] = mw == m ? 1.0f : __builtin_amdgcn_exp2f(mw - m);
      l_run += f[w] * stats[1][w][row];
    }
    float o[8] = {};
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      const uint8_t* part = lds + w * 2 * T;
      const f32x4 lo = *reinterpret_cast<const f32x4*>(part + part_off(row, 2 * ch));
      const f32x4 hi = *reinterpret_cast<const f32x4*>(part + part_off(row, 2 * ch + 1));
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        o[e] = fmaf(f[w], lo[e], o[e]);
        o[4 + e] = fmaf(f[w], hi[e], o[4 + e]);
      }
    }
    if (p.splits > 1) {
      const int64_t at = static_cast<int64_t>(s.unit) * p.rows + s.row0 + row;
      if (ch == 0) *reinterpret_cast<float2*>(p.part_ml + at * 2) = make_float2(m, l_run);
      *reinterpret_cast<f32x4*>(p.part_o + at * D + ch * 8) = f32x4{o[0], o[1], o[2], o[3]};
      *reinterpret_cast<f32x4*>(p.part_o + at * D + ch * 8 + 4) = f32x4{o[4], o[5], o[6], o[7]};
      continue;
    }
    int64_t o_at, lse_at;
    if (!out_row(p, s, s.row0 + row, written, o_at, lse_at)) continue;
    if (add) add_infinite<E>(p, s.b, s.head, (s.row0 + row) % p.n_q, ch, o);
    *reinterpret_cast<u32x4*>(p.o + o_at + ch * 8) = pack8<E>(o, inverse_sum(l_run));
    if (p.lse != nullptr && ch == 0) p.lse[lse_at] = lse_of(m, l_run);
  }
}

// Lanes of a join kernel: D / 8 for a row's values, times the groups that its splits are dealt to
// (a power of two; all of a row's lanes lie in one wave).
template <int D>
struct JoinLanes {
  static constexpr int kLanes = D / 8, kMost = 64 / kLanes;
  int64_t row;
  int ch, group, groups;
  __device__ __forceinline__ JoinLanes(uint32_t block, int n_groups) : groups(n_groups) {
    const int64_t i = static_cast<int64_t>(block) * 256 + threadIdx.x;
    const int64_t all = i / kLanes;
    ch = static_cast<int>(i % kLanes);
    group = static_cast<int>(all & (groups - 1));
    row = all / groups;
  }
  // over the groups, the same in all of them
  template <class F>
  __device__ __forceinline__ float reduce(float v, F f) const {
    for (int d = kLanes; d < kLanes * groups; d *= 2) v = f(v, __shfl_xor(v, d, 64));
    return v;
  }
  // Groups for few rows, whose lanes alone would not fill the chip: 256 rows of 8 splits, 128 heads:
  // 8.9 us in one group, 4.4 in four; 16384 rows of 4 splits: 7.9 and 13.6.
  static int groups_of(int64_t rows, int splits) {
    int n = 1;
    while (n < kMost && n < splits && rows * kLanes * n * 2 <= 65536) n *= 2;
    return n;
  }
};

// Adds up the splits of a row, relative to the largest reference point.
template <int D, class E>
__device__ __forceinline__ void kv_join_body(const KvArgs& p) {
  const JoinLanes<D> at(blockIdx.x, p.join_groups);
  const int64_t bh = at.row / p.rows;
  const int row = static_cast<int>(at.row - bh * p.rows);
  Share s;
  s.b = static_cast<int>(bh / p.kv_heads);
  s.head = static_cast<int>(bh - static_cast<int64_t>(s.b) * p.kv_heads);
  if (s.b >= p.batch) return;
  int64_t o_at, lse_at;
  if (!out_row(p, s, row, written_of(p, s.b), o_at, lse_at)) return;  // all lanes of the row
  const int64_t first = static_cast<int64_t>(s.b) * p.splits * p.kv_heads + s.head;  // unit of split 0
  float m = -INFINITY;
  int add = 0;
#pragma unroll 4
  for (int k = at.group; k < p.splits; k += at.groups) {
    const int64_t unit = first + static_cast<int64_t>(k) * p.kv_heads;
    m = fmaxf(m, p.part_ml[(unit * p.rows + row) * 2]);
    if (p.k_draft) add |= p.infinite[unit];
  }
  m = at.reduce(m, [](float a, float b) { return fmaxf(a, b); });
  float l_run = 0.f, o[8] = {};
#pragma unroll 4
  for (int k = at.group; k < p.splits; k += at.groups) {
    const int64_t part = (first + static_cast<int64_t>(k) * p.kv_heads) * p.rows + row;
    const float2 ml = *reinterpret_cast<const float2*>(p.part_ml + part * 2);
    const f32x4 lo = *reinterpret_cast<const f32x4*>(p.part_o + part * D + at.ch * 8);
    const f32x4 hi = *reinterpret_cast<const f32x4*>(p.part_o + part * D + at.ch * 8 + 4);
    const float f = ml.x == m ? 1.0f : __builtin_amdgcn_exp2f(ml.x - m);
    const bool keys = ml.y != 0.f;  // without any, its part is not written
    l_run += keys ? f * ml.y : 0.f;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      o[e] = fmaf(f, keys ? lo[e] : 0.f, o[e]);
      o[4 + e] = fmaf(f, keys ? hi[e] : 0.f, o[4 + e]);
    }
  }
  const auto sum = [](float a, float b) { return a + b; };
  l_run = at.reduce(l_run, sum);
#pragma unroll
  for (int e = 0; e < 8; ++e) o[e] = at.reduce(o[e], sum);
  const bool any = at.reduce(add ? 1.0f : 0.0f, sum) != 0.f;
  if (at.group != 0) return;
  if (any) add_infinite<E>(p, s.b, s.head, row % p.n_q, at.ch, o);
  *reinterpret_cast<u32x4*>(p.o + o_at + at.ch * 8) = pack8<E>(o, inverse_sum(l_run));
  if (p.lse != nullptr && at.ch == 0) p.lse[lse_at] = lse_of(m, l_run);
}

}  // namespace kv
}  // namespace asc
